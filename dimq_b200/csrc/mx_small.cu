// The microscaled 4-bit product for a few rows of x (single tokens): one launch, x quantised on the way.
//
// What bounds it is reading the weight, so the weight is the wide operand: a block takes 128 of its rows as the lanes of
// the block-scaled MMA (kind::mxf4, see mx_gemm.cu) and the rows of x as its columns, and a cluster of blocks divides k.
// Every block fires all its copies at once - codes and scales of its slice, up to 102 KB - and quantises its slice of x
// while they come; then a few MMAs, and the cluster adds its partial sums over distributed shared memory, in rank order,
// each block finishing a share of the rows.
#include "mx_tile.cuh"

namespace dimq {
namespace {

using namespace mx;

constexpr int kThreads = 256;
constexpr int kMostSteps = 6;                 // 256-k steps a block holds
constexpr int kMostSlices = 8;                // blocks of a cluster
// Tensor-memory columns of a block, 32 of sums and 16 of scales per step, in powers of two.  A block that waits for columns
// keeps its cluster waiting, and so the columns that its peers hold: the blocks that fit on an SM must never want more than
// its 512.  So a block asks for at least as much shared memory (28.5 KB for every 64 columns) as makes that so for any mix.
__host__ __device__ constexpr uint32_t columns_of(int room) { return room <= 2 ? 64u : 128u; }
constexpr size_t kBytesPer64Columns = 28 * 1024 + 512;

struct SmallParams {
  const void* x;
  const uint8_t* sfa;
  Out out;                                    // rows = M, cols = N
  int64_t K;
  int k_tiles, steps, slices;                 // scale tiles along k, 256-k steps, blocks of a cluster
  int room;                                   // steps a block has room for
};

struct SmallHeader {
  uint64_t full, done;
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float peer_float(uint32_t addr, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
}

// bytes of a 256-k step: 128 weight rows, their scales, NB rows of x, theirs
constexpr uint32_t step_bytes(int nb) { return 128u * 128u + 1024u + static_cast<uint32_t>(nb) * 128u + 1024u; }

template <int NB, typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
mx_small_kernel(const __grid_constant__ CUtensorMap codes, const SmallParams p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  // [step: weight codes][step: weight scales][step: x codes][step: x scales][sums NB x 128][header], all by steps of room
  unsigned char* s_sfa = smem + p.room * 16384;
  unsigned char* s_x = s_sfa + p.room * 1024;
  unsigned char* s_sfx = s_x + p.room * (NB * 128);
  float* s_sum = reinterpret_cast<float*>(s_sfx + p.room * 1024);
  SmallHeader* hdr = reinterpret_cast<SmallHeader*>(s_sum + NB * 128);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slices = p.slices, rank = slices > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int row_tile = static_cast<int>(blockIdx.x) / slices;
  const int step0 = p.steps * rank / slices, n_steps = p.steps * (rank + 1) / slices - step0;   // >= 1: slices <= steps
  const int tiles_here = min(2 * n_steps, p.k_tiles - 2 * step0);

  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&hdr->full), 1);
    mbar_init(smem_u32(&hdr->done), 1);
    hdr->abort_flag = 0u;
    fence_barrier_init();
  }
  __syncwarp();
  if (warp == 0) {
    if (elect_one()) {      // the whole slice of the weight at once
      const uint32_t full = smem_u32(&hdr->full);
      mbar_arrive_expect_tx(full, static_cast<uint32_t>(n_steps) * 16384u + static_cast<uint32_t>(tiles_here) * kTileBytes);
      for (int i = 0; i < n_steps; ++i) tma_load_2d(smem_u32(smem + i * 16384), &codes, full, (step0 + i) * 128, row_tile * 128);
      bulk_load(smem_u32(s_sfa), p.sfa + (static_cast<int64_t>(row_tile) * p.k_tiles + 2 * step0) * kTileBytes,
                static_cast<uint32_t>(tiles_here) * kTileBytes, full);
    }
    __syncwarp();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&hdr->tmem_base), columns_of(p.room));
    tmem_relinquish();
  }

  // this slice of x: four lanes hold a block of 32, eight values each
  {
    const int blocks = tiles_here * 4, rows = static_cast<int>(p.out.rows);
    const int units = rows * blocks;
    const T* x = static_cast<const T*>(p.x);
    for (int u0 = warp * 8; u0 < units; u0 += kThreads / 4) {
      const int u = u0 + (lane >> 2);
      const int r = min(u / blocks, rows - 1), b = u - (u / blocks) * blocks;
      const int64_t k = static_cast<int64_t>(step0) * 256 + b * 32 + (lane & 3) * 8;
      float v[8];
      load8<T, VEC>(x + r * p.K, k, p.K, v);
      const uint32_t byte = scale_byte(block_top(v), 2);
      if (u < units) {
        const int step = b >> 3, piece = b & 7;      // 16 bytes of codes: piece of the step's 128-byte row, swizzled
        *reinterpret_cast<uint32_t*>(s_x + step * (NB * 128) + r * 128 + ((piece ^ (r & 7)) << 4) + (lane & 3) * 4) = encode_fp4(v, byte);
        if ((lane & 3) == 0) s_sfx[step * 1024 + ((b >> 2) & 1) * kTileBytes + r * 16 + (b & 3)] = static_cast<uint8_t>(byte);
      }
    }
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = hdr->tmem_base;
  bool ok = true;
  if (warp == 0) {
    ok = __all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&hdr->full), 0u, &hdr->abort_flag, 0x4100u));
    if (ok) {
      if (elect_one()) {
        const uint64_t sfa0 = scale_desc(smem_u32(s_sfa)), sfx0 = scale_desc(smem_u32(s_sfx));
        for (int t = 0; t < tiles_here; ++t) {
          copy_scales(tmem + 32 + 8 * t, sfa0 + static_cast<uint64_t>(t * (kTileBytes >> 4)));
          copy_scales(tmem + 36 + 8 * t, sfx0 + static_cast<uint64_t>(t * (kTileBytes >> 4)));
        }
        for (int t = 0; t < tiles_here; ++t) {
          const uint64_t a = make_smem_desc_sw128(smem_u32(smem + (t >> 1) * 16384)) + static_cast<uint64_t>(4 * (t & 1));
          const uint64_t b = make_smem_desc_sw128(smem_u32(s_x + (t >> 1) * (NB * 128))) + static_cast<uint64_t>(4 * (t & 1));
#pragma unroll
          for (int j = 0; j < 2; ++j)
            mma_mxf4(tmem, a + 2 * j, b + 2 * j, mxf4_idesc(128, NB, j), tmem + 32 + 8 * t, tmem + 36 + 8 * t, (t | j) ? 1u : 0u);
        }
        mma_commit(smem_u32(&hdr->done));
      }
    } else {                // gave up: bounded wait for the copies in flight
      for (uint32_t it = 0; it < kSpinLimit; ++it)
        if (mbar_try_wait(smem_u32(&hdr->full), 0u)) break;
    }
    __syncwarp();
  }
  if (warp < 4) {
    ok = __all_sync(0xFFFFFFFFu, ok && mbar_wait(smem_u32(&hdr->done), 0u, &hdr->abort_flag, 0x4200u));
    tc_fence_after();
    if (ok) {
      const uint32_t at = tmem + (static_cast<uint32_t>(warp * 32) << 16);
#pragma unroll
      for (int c = 0; c < NB / 8; ++c) {
        uint32_t r[8];
        tmem_ld8(at + 8 * c, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 8; ++j) s_sum[(8 * c + j) * 128 + warp * 32 + lane] = __uint_as_float(r[j]);
      }
    }
  }
  tc_fence_before();
  if (slices > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  // each block finishes a share of the weight rows
  const int share = 128 / slices;
  const int64_t n_first = static_cast<int64_t>(row_tile) * 128 + rank * share;
  for (int i = threadIdx.x; i < static_cast<int>(p.out.rows) * share; i += kThreads) {
    const int m = i / share, c = i - m * share;
    const int64_t n = n_first + c;
    if (n >= p.out.cols) continue;
    const int at = m * 128 + rank * share + c;
    float s;
    if (slices > 1) {
      const uint32_t addr = smem_u32(s_sum + at);
      float part[kMostSlices];
#pragma unroll
      for (int r = 0; r < kMostSlices; ++r) part[r] = r < slices ? peer_float(addr, static_cast<uint32_t>(r)) : 0.0f;
      s = part[0];
#pragma unroll
      for (int r = 1; r < kMostSlices; ++r)
        if (r < slices) s += part[r];
    } else {
      s = s_sum[at];
    }
    if (p.out.bias != nullptr) s += load_as_float(p.out.bias, p.out.bias_dtype, n);
    const int64_t o = m * p.out.cols + n;
    const float res = p.out.residual != nullptr ? load_as_float(p.out.residual, p.out.dtype, o) : 0.0f;
    store_from_float(p.out.y, p.out.dtype, o, activate_any(s, res, p.out.epilogue));
  }
  if (slices > 1) {         // no block leaves while a peer may read its sums
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, columns_of(p.room));
  }
}

template <int NB, typename T>
int launch_small(const CUtensorMap& codes, const SmallParams& p, bool vec, int64_t row_blocks, cudaStream_t st) {
  size_t smem = 1024 + p.room * step_bytes(NB) + NB * 512 + 64;
  const size_t least = columns_of(p.room) / 64 * kBytesPer64Columns;
  if (smem < least) smem = least;
  auto kern = vec ? mx_small_kernel<NB, T, true> : mx_small_kernel<NB, T, false>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemMax));
  if (e != cudaSuccess) return static_cast<int>(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(row_blocks * p.slices));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(p.slices);
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, codes, p);
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
}

template <typename T>
int small_as(const CUtensorMap& codes, const SmallParams& p, bool vec, int64_t row_blocks, cudaStream_t st) {
  if (p.out.rows <= 8) return launch_small<8, T>(codes, p, vec, row_blocks, st);
  return launch_small<16, T>(codes, p, vec, row_blocks, st);
}

}  // namespace

bool mx_small_takes(int64_t M, int64_t N, int64_t K) {
  return M <= 16 && (mx::block_tiles(K) + 1) / 2 <= kMostSteps * kMostSlices && mx::row_tiles(N) <= 0x7FFFFFFF / kMostSlices;
}

int mx_small(const void* x, int x_dtype, const uint8_t* wc, const uint8_t* ws, const void* bias, int bias_dtype, const void* residual,
             void* y, int y_dtype, int64_t M, int64_t N, int64_t K, int epilogue, cudaStream_t st) {
  SmallParams p = {};
  p.x = x;
  p.sfa = ws;
  p.out = {y, residual, bias, M, N, bias_dtype, y_dtype, epilogue, 0};
  p.K = K;
  p.k_tiles = static_cast<int>(block_tiles(K));
  p.steps = (p.k_tiles + 1) / 2;
  const int64_t row_blocks = row_tiles(N);
  int slices = 1;
  while (slices < kMostSlices && 2 * slices <= p.steps && (row_blocks * slices < 2 * kNumSMs || (p.steps + slices - 1) / slices > kMostSteps)) slices *= 2;
  p.slices = slices;
  p.room = (p.steps + slices - 1) / slices;
  CUtensorMap codes;
  if (!code_map(&codes, wc, N, K, 128)) return DIMQ_ERR_DRIVER;
  const bool vec = aligned(x, 16) && (K * dtype_size(x_dtype)) % 16 == 0;
  if (x_dtype == DIMQ_F32) return small_as<float>(codes, p, vec, row_blocks, st);
  if (x_dtype == DIMQ_F16) return small_as<__half>(codes, p, vec, row_blocks, st);
  return small_as<__nv_bfloat16>(codes, p, vec, row_blocks, st);
}

int read_mx_small_status(uint32_t* status) { return tc::read_and_clear_device_status(status); }

}  // namespace dimq
