// What the microscaled products share: copies, the output of a 32 x 32 piece, the tensor-map encoder.
#pragma once

#include "mx_common.cuh"
#include "tc_common.cuh"

namespace dimq {
namespace mx {

using namespace tc;

constexpr int kHeaderBytes = 1024;
constexpr int kEpiWarps = 8;
constexpr size_t kSmemMax = 227 * 1024;   // what a block may use: every kernel's limit is set to this, never to a call's own size

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_tiled() {
  static EncodeTiledFn fn = [] {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &qres) == cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      return reinterpret_cast<EncodeTiledFn>(sym);
    return static_cast<EncodeTiledFn>(nullptr);
  }();
  return fn;
}

// rank 2 or 3, innermost first; zero fill outside
inline bool encode_map(CUtensorMap* m, CUtensorMapDataType type, int rank, const void* base, const cuuint64_t* dims,
                       const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle) {
  EncodeTiledFn encode = encode_tiled();
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return encode != nullptr &&
         encode(m, type, static_cast<cuuint32_t>(rank), const_cast<void*>(base), dims, strides, box, estr,
                CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

inline CUtensorMapDataType map_dtype(int dtype) {
  return dtype == DIMQ_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                           : dtype == DIMQ_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// Launched as a programmatic dependent: the prologue overlaps the end of the kernel before it in the stream; every thread
// of such a kernel waits (wait_for_inputs) before it touches global memory.
template <typename Kern, typename... Args>
cudaError_t launch_dependent(Kern kern, unsigned grid, int threads, size_t smem, cudaStream_t st, int cluster, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

#ifdef __CUDACC__

__device__ __forceinline__ void wait_for_inputs() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar) : "memory");
}

// scale tile (32 rows x 16 bytes) -> 4 columns, the same in all four lane quarters.  PAIR: in both blocks, each from its
// own shared memory
template <bool PAIR = false>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t desc) {
  if (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// rows of 16 bytes, eight to a 128-byte group, no swizzle
__device__ __forceinline__ uint64_t scale_desc(uint32_t smem) {
  return static_cast<uint64_t>((smem & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(128 >> 4) << 16) |
         (static_cast<uint64_t>(128 >> 4) << 32) | (static_cast<uint64_t>(1) << 46);
}
template <bool PAIR = false>
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t accumulate) {
  if (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// e2m1 times e2m1 with e8m0 scales; `half`: which two of the four scale bytes of a column belong to this step
__device__ constexpr uint32_t mxf4_idesc(int m, int n, int half) {
  return (static_cast<uint32_t>(2 * half) << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) |
         (static_cast<uint32_t>(m >> 7) << 27) | (static_cast<uint32_t>(2 * half) << 29);
}

// ---- clusters: few-row products divide k over one, large tiles are shared by two blocks (no multicast copies) ----
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t map_to_cta(uint32_t addr, uint32_t rank) {   // the same shared address in another block
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
__device__ __forceinline__ void remote_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const void* tmap, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t smem_dst, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void commit(uint32_t bar) {   // PAIR: one arrival in both blocks
  if (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
  else
    mma_commit(bar);
}

// A block that gave up a wait must not leave while copies into its shared memory are under way.  Its producers note how often
// they filled each stage; when all warps have stopped, one thread waits (together no longer than one more limit) for the last
// filling of each.  PAIR: the first block's barriers count both blocks' copies, so it waits for both; a filling that only one
// of the two began never completes and is waited for as long as the limit allows.
__device__ __forceinline__ uint32_t peer_word(const uint32_t* at, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(map_to_cta(smem_u32(at), rank)) : "memory");
  return v;
}
template <bool PAIR>
__device__ __forceinline__ void wait_for_copies(const uint64_t* full, const uint32_t* filled, uint32_t stages) {
  uint32_t left = kSpinLimit;
  for (uint32_t s = 0; s < stages; ++s) {
    uint32_t n = filled[s];
    if (PAIR) n = max(n, peer_word(filled + s, 1));
    while (n != 0u && left != 0u && !mbar_try_wait(smem_u32(full + s), (n - 1u) & 1u)) --left;
  }
}
// The end of a block of the persistent kernels, all threads: whether anyone gave up (PAIR: in either block) decides alike for
// all, and no block of a pair leaves while the other may use its memories.
template <bool PAIR>
__device__ __forceinline__ void leave_together(volatile uint32_t* abort_flag, const uint64_t* full, const uint32_t* filled, uint32_t stages,
                                               int rank) {
  __syncthreads();
  if constexpr (PAIR) {
    if (threadIdx.x == 0 && *abort_flag != 0u)
      asm volatile("st.shared::cluster.u32 [%0], %1;"
                   ::"r"(map_to_cta(smem_u32(const_cast<const uint32_t*>(abort_flag)), static_cast<uint32_t>(rank ^ 1))), "r"(1u) : "memory");
    __syncwarp();             // the cluster's barrier wants whole warps
    cluster_arrive();
    cluster_wait();
  }
  if (*abort_flag == 0u) return;
  if (threadIdx.x == 0 && rank == 0) wait_for_copies<PAIR>(full, filled, stages);
  __syncwarp();
  if constexpr (PAIR) { cluster_arrive(); cluster_wait(); }
  else __syncthreads();
}

// One lane of an epilogue warp whose sums are in registers: the last of the warps hands the accumulator back (PAIR: to the
// first block's barrier).  Nothing waits here: with two accumulators the warps need not keep step (a barrier among them held
// the fp32 8192 x 11008 -> 4096 weight gradient at 630 us, 540 so).
template <bool PAIR>
__device__ __forceinline__ void hand_back(uint32_t* count, uint32_t bar) {
  __threadfence_block();
  if (atomicAdd(count, 1u) == kEpiWarps - 1) {
    *count = 0u;
    __threadfence_block();
    if (PAIR) remote_arrive(map_to_cta(bar, 0));
    else mbar_arrive(bar);
  }
}

// Whether all of a barrier's `threads` (whole warps) say yes
__device__ __forceinline__ bool all_agree(int id, int threads, bool yes) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(r) : "r"(static_cast<uint32_t>(yes)), "r"(id), "r"(threads) : "memory");
  return r != 0u;
}

__device__ __forceinline__ float max_nan(float a, float b) {   // a NaN stays one
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// GELU of a result in 16 bits takes the polynomial error function (1.5e-7 of v, in the tail most of GELU: at v = -5, 4 %); of
// one in fp32 the complementary error function, good to a few steps in relative terms wherever GELU is a normal number.
__device__ __forceinline__ float gelu_fast(float v) { return 0.5f * v * (1.0f + fast_erf(v * 0.70710678118654752440f)); }
__device__ __forceinline__ float gelu_wide(float v) { return 0.5f * v * erfcf(v * -0.70710678118654752440f); }

// RELU, ADD_RELU or none
__device__ __forceinline__ float activate_linear(float v, float res, int epilogue) {
  if (epilogue == DIMQ_EPI_NONE) return v + res;
  return epilogue == DIMQ_EPI_ADD_RELU ? max_nan(v + res, 0.0f) : max_nan(v, 0.0f) + res;
}
template <bool WIDE>
__device__ __forceinline__ float activate_any(float v, float res, int epilogue) {
  if (epilogue == DIMQ_EPI_GELU) return (WIDE ? gelu_wide(v) : gelu_fast(v)) + res;
  return activate_linear(v, res, epilogue);
}

struct Out {            // where a product goes
  void* y;
  const void* residual; // y's type and layout, or null
  const void* bias;     // one per column, or null
  int64_t rows, cols;
  int bias_dtype, dtype, epilogue;
  int tma;              // rows of whole 16-byte pieces: the tensor map stores them
};

template <int ES>
__device__ __forceinline__ float element(const uint4& q, int i, int dtype) {
  const uint32_t w = i < (ES == 2 ? 2 : 1) ? q.x : i < (ES == 2 ? 4 : 2) ? q.y : i < (ES == 2 ? 6 : 3) ? q.z : q.w;
  if (ES == 4) return __uint_as_float(w);
  const unsigned short h = static_cast<unsigned short>(i & 1 ? w >> 16 : w);
  return dtype == DIMQ_BF16 ? __uint_as_float(static_cast<uint32_t>(h) << 16) : __half2float(__ushort_as_half(h));
}

// Shared memory of an epilogue warp: two pieces of 2 KB that map stores read in turn (16-bit results), or one of 4 KB
// (fp32: a second one would cost the ring a stage).
constexpr uint32_t kStagingBytes = 4096;

// Sums of 32 rows x 32 columns (lane = row, v = its columns from n0 on) -> y.  bias: 32 floats in shared memory, or null.
// stage: this warp's shared memory, 1024-aligned; turn: which piece is next.
// With a map: bias, activation and residual on the lane's row, packed into the swizzled box the map stores.  Without: the
// sums change hands through shared memory, so that a warp stores 32 neighbours of one row at a time.  (Boxes of 64 columns,
// and 16-byte stores of four rows at a time instead of the map, were slower: 25216 x 768 -> 2304 bf16 59 and 69 us against
// 57.)
// GELU of fp32 is done in the box, four values at a time: unrolled over the row in registers it would not fit.  It costs the
// instructions of erfc: 2048 x 1024 -> 4096 35.6 us (the polynomial 28.9, ReLU 15.0; 8 and 16 values at a time 37 and 39).
// (ACT: whether there can be an activation.)
template <int ES, bool ACT = true>
__device__ __forceinline__ void put_chunk(float (&v)[32], const Out& o, const CUtensorMap* map, unsigned char* stage, uint32_t& turn,
                                          const float* bias, int64_t row0, int64_t n0, int lane) {
  if (o.tma) {
    const int64_t row = row0 + lane;
    if (bias != nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 b = *reinterpret_cast<const float4*>(bias + 4 * j);   // one address for all lanes
        v[4 * j] += b.x; v[4 * j + 1] += b.y; v[4 * j + 2] += b.z; v[4 * j + 3] += b.w;
      }
    }
    const bool in_box = ES == 4 && ACT && o.epilogue == DIMQ_EPI_GELU;
    if (o.residual != nullptr && !in_box) {
      constexpr int kPer = 16 / ES;
      const char* r = static_cast<const char*>(o.residual) + (row * o.cols + n0) * ES;
#pragma unroll
      for (int c = 0; c < 32 / kPer; ++c) {
        uint4 q = make_uint4(0u, 0u, 0u, 0u);
        if (row < o.rows && n0 + c * kPer < o.cols) q = __ldg(reinterpret_cast<const uint4*>(r) + c);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const float res = element<ES>(q, i, o.dtype);
          v[c * kPer + i] = ES == 2 ? activate_any<false>(v[c * kPer + i], res, o.epilogue) : activate_linear(v[c * kPer + i], res, o.epilogue);
        }
      }
    } else if (o.epilogue == DIMQ_EPI_GELU) {
      if (ES == 2) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = gelu_fast(v[j]);
      }
    } else if (o.epilogue != DIMQ_EPI_NONE) {
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = max_nan(v[j], 0.0f);
    }
    if (ES == 2) {
      stage += turn * 2048;
      turn ^= 1u;
      if (elect_one()) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");   // the store before the last has read this piece
    } else if (elect_one()) {
      tma_store_wait_read();
    }
    __syncwarp();
    if (ES == 2) {   // 64-byte rows, 64-byte swizzle
      unsigned char* p = stage + lane * 64;
      const int sw = (lane >> 1) & 3;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = v[8 * j + 2 * i], b = v[8 * j + 2 * i + 1];
          if (o.dtype == DIMQ_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(b), "f"(a));
          else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(b), "f"(a));
        }
        *reinterpret_cast<uint4*>(p + ((j ^ sw) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    } else {         // 128-byte rows, 128-byte swizzle
      unsigned char* p = stage + lane * 128;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        *reinterpret_cast<float4*>(p + ((j ^ (lane & 7)) << 4)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
      if (in_box) {
        const float* r = static_cast<const float*>(o.residual) + row * o.cols + n0;
#pragma unroll 1
        for (int j = 0; j < 8; ++j) {   // the lane's own row
          float4* at = reinterpret_cast<float4*>(p + ((j ^ (lane & 7)) << 4));
          float4 q = make_float4(0.0f, 0.0f, 0.0f, 0.0f), g = *at;
          if (o.residual != nullptr && row < o.rows && n0 + 4 * j < o.cols) q = __ldg(reinterpret_cast<const float4*>(r) + j);
          g.x = gelu_wide(g.x) + q.x; g.y = gelu_wide(g.y) + q.y; g.z = gelu_wide(g.z) + q.z; g.w = gelu_wide(g.w) + q.w;
          *at = g;
        }
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (elect_one()) {
      tma_store_2d(map, smem_u32(stage), static_cast<int>(n0), static_cast<int>(row0));
      tma_store_commit();
    }
    __syncwarp();
    return;
  }
  float* f = reinterpret_cast<float*>(stage);
  if (elect_one()) tma_store_wait_read();   // pieces stored through a map before this one
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 32; ++j) f[lane * 32 + (j ^ lane)] = v[j];
  __syncwarp();
  const int64_t n = n0 + lane;
  const float b = bias != nullptr ? bias[lane] : 0.0f;
  if (n < o.cols) {
    const int rows = static_cast<int>(o.rows - row0 < 32 ? o.rows - row0 : 32);
    if (ES == 4 && ACT && o.epilogue == DIMQ_EPI_GELU) {   // apart: it is long
#pragma unroll 4
      for (int r = 0; r < rows; ++r) {
        const int64_t at = (row0 + r) * o.cols + n;
        const float res = o.residual != nullptr ? static_cast<const float*>(o.residual)[at] : 0.0f;
        static_cast<float*>(o.y)[at] = gelu_wide(f[r * 32 + (lane ^ r)] + b) + res;
      }
    } else {
#pragma unroll 4
      for (int r = 0; r < rows; ++r) {
        const int64_t at = (row0 + r) * o.cols + n;
        const float res = o.residual != nullptr ? load_as_float(o.residual, o.dtype, at) : 0.0f;
        const float v = f[r * 32 + (lane ^ r)] + b;
        store_from_float(o.y, o.dtype, at, ES == 2 && ACT ? activate_any<false>(v, res, o.epilogue) : activate_linear(v, res, o.epilogue));
      }
    }
  }
  __syncwarp();
}

#endif

// codes of a 4-bit matrix, boxes of 128 bytes (256 values) x box_rows
inline bool code_map(CUtensorMap* m, const void* codes, int64_t rows, int64_t K, int box_rows) {
  const cuuint64_t pitch = static_cast<cuuint64_t>(codes_pitch(K, DIMQ_MX_FP4));
  const cuuint64_t dims[2] = {pitch, static_cast<cuuint64_t>(rows)};
  const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)};
  return encode_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, codes, dims, &pitch, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

inline bool out_by_map(const Out& o) {
  const int64_t es = o.dtype == DIMQ_F32 ? 4 : 2;
  return aligned(o.y, 16) && (o.residual == nullptr || aligned(o.residual, 16)) && (o.cols * es) % 16 == 0;
}
inline bool encode_out(CUtensorMap* m, const Out& o) {   // boxes of 32 rows x 32 columns
  const cuuint64_t es = o.dtype == DIMQ_F32 ? 4 : 2;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(o.cols), static_cast<cuuint64_t>(o.rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(o.cols) * es};
  const cuuint32_t box[2] = {32, 32};
  return encode_map(m, map_dtype(o.dtype), 2, o.y, dims, strides, box, es == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

}  // namespace mx
}  // namespace dimq
