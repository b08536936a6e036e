// The microscaled 4-bit product for a few rows of x (single tokens): one launch, x quantised on the way.
//
// What bounds it is reading the weight, so the weight is the wide operand: a block takes 128 of its rows as the lanes of
// the block-scaled MMA (kind::mxf4, see mx_gemm.cu) and the rows of x as its columns, and a cluster of blocks divides k.
// A block starts as many copies as its ring holds before it looks at x, and quantises its slice of x while they come; then
// steps of 256 k go through the ring, and the cluster adds its partial sums over distributed shared memory, in rank order,
// each block finishing a share of the rows.
#include "mx_tile.cuh"

namespace dimq {
namespace {

using namespace mx;

constexpr int kThreads = 256;
constexpr int kMostSteps = 16;                // 256-k steps of a block (their x is kept whole)
constexpr int kMostSlices = 8;                // blocks of a cluster
constexpr int kMostStages = 6;
constexpr uint32_t kWeightBytes = 128 * 128 + 1024;   // a ring stage: the codes of 128 rows x 256 k, and their scales
// Tensor-memory columns of a block: 32 of sums and 16 of scales per ring stage, a power of two.  A block that waits for
// columns keeps its cluster waiting, and so the columns that its peers hold: the blocks that fit on an SM must never want
// more than its 512.  So a block asks for at least as much shared memory (28.5 KB for every 64 columns) as makes that so
// for any mix of such blocks.
__host__ __device__ constexpr uint32_t columns_of(int stages) { return stages <= 2 ? 64u : 128u; }
constexpr size_t kBytesPer64Columns = 28 * 1024 + 512;

struct SmallParams {
  const void* x;
  const uint8_t* sfa;
  Out out;                                    // rows = M, cols = N
  int64_t K;
  int k_tiles, steps, slices;                 // scale tiles along k, 256-k steps, blocks of a cluster
  int room, stages;                           // steps a block has room for x of, ring stages
};

struct SmallHeader {
  uint64_t full[kMostStages], empty[kMostStages], done;
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
};

__device__ __forceinline__ float peer_float(uint32_t addr, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_cta(addr, rank)) : "memory");
  return v;
}
template <typename T>
__device__ __forceinline__ Eight<T> load_single(const T* __restrict__ row, int64_t k, int64_t cols) {
  Eight<T> e = no_values<T>();
  T* v = reinterpret_cast<T*>(e.w);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k + i < cols) v[i] = row[k + i];
  return e;
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
}

template <int NB, typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
mx_small_kernel(const __grid_constant__ CUtensorMap codes, const SmallParams p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  // [stage: weight codes, scales][step: x codes][step: x scales][sums NB x 128][header]
  unsigned char* s_x = smem + p.stages * kWeightBytes;
  unsigned char* s_sfx = s_x + p.room * (NB * 128);
  float* s_sum = reinterpret_cast<float*>(s_sfx + p.room * 1024);
  SmallHeader* hdr = reinterpret_cast<SmallHeader*>(s_sum + NB * 128);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slices = p.slices, rank = slices > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int row_tile = static_cast<int>(blockIdx.x) / slices;
  const int step0 = p.steps * rank / slices, n_steps = p.steps * (rank + 1) / slices - step0;   // >= 1: slices <= steps
  const int tiles_here = min(2 * n_steps, p.k_tiles - 2 * step0);

  if (threadIdx.x == 0) {
    for (int i = 0; i < kMostStages; ++i) { mbar_init(smem_u32(&hdr->full[i]), 1); mbar_init(smem_u32(&hdr->empty[i]), 1); }
    mbar_init(smem_u32(&hdr->done), 1);
    hdr->abort_flag = 0u;
    fence_barrier_init();
    prefetch_tensormap(&codes);
  }
  __syncwarp();
  const auto load_step = [&](int i, int stage) {   // one lane
    const uint32_t full = smem_u32(&hdr->full[stage]), dst = smem_u32(smem + stage * kWeightBytes);
    const uint32_t sf = static_cast<uint32_t>(min(2, tiles_here - 2 * i)) * kTileBytes;
    mbar_arrive_expect_tx(full, 16384u + sf);
    tma_load_2d(dst, &codes, full, (step0 + i) * 128, row_tile * 128);
    bulk_load(dst + 16384, p.sfa + (static_cast<int64_t>(row_tile) * p.k_tiles + 2 * (step0 + i)) * kTileBytes, sf, full);
  };
  wait_for_inputs();
  if (warp == 0) {
    if (elect_one())
      for (int i = 0; i < p.stages && i < n_steps; ++i) load_step(i, i);
    __syncwarp();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&hdr->tmem_base), columns_of(p.stages));
    tmem_relinquish();
  }

  // this slice of x: four lanes hold a block of 32, eight values each; kAhead blocks' loads in flight
  {
    constexpr int kAhead = 4;
    const int blocks = tiles_here * 4, rows = static_cast<int>(p.out.rows);
    const int units = rows * blocks;
    const T* x = static_cast<const T*>(p.x);
    for (int u0 = warp * 8; u0 < units; u0 += kAhead * (kThreads / 4)) {
      Eight<T> v[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int u = min(u0 + i * (kThreads / 4) + (lane >> 2), units - 1), r = u / blocks;
        const int64_t k = static_cast<int64_t>(step0) * 256 + (u - r * blocks) * 32 + (lane & 3) * 8;
        v[i] = VEC ? load_pieces<T>(x + r * p.K, k, p.K) : load_single<T>(x + r * p.K, k, p.K);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int u = u0 + i * (kThreads / 4) + (lane >> 2), r = u / blocks, b = u - r * blocks;
        const uint32_t byte = scale_byte(block_top(v[i]), 2);
        if (u < units) {
          const int step = b >> 3, piece = b & 7;    // 16 bytes of codes: piece of the step's 128-byte row, swizzled
          *reinterpret_cast<uint32_t*>(s_x + step * (NB * 128) + r * 128 + ((piece ^ (r & 7)) << 4) + (lane & 3) * 4) = encode_fp4(v[i], byte);
          if ((lane & 3) == 0) s_sfx[step * 1024 + ((b >> 2) & 1) * kTileBytes + r * 16 + (b & 3)] = static_cast<uint8_t>(byte);
        }
      }
    }
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  let_dependents_start();       // every block of this grid runs by now and has its columns
  const uint32_t tmem = hdr->tmem_base;
  bool ok = true;
  int fetched = n_steps < p.stages ? n_steps : p.stages;   // warp 1: steps whose copies have been issued
  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    for (int i = 0; i < n_steps; ++i) {
      if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&hdr->full[stage]), phase, &hdr->abort_flag, 0x4100u | stage))) { ok = false; break; }
      if (elect_one()) {
        const uint32_t w = smem_u32(smem + stage * kWeightBytes), sfa = tmem + 32 + 16 * stage, sfx = sfa + 8;
        const uint64_t sfa0 = scale_desc(w + 16384), sfx0 = scale_desc(smem_u32(s_sfx + i * 1024));
        const uint64_t a0 = make_smem_desc_sw128(w), b0 = make_smem_desc_sw128(smem_u32(s_x + i * (NB * 128)));
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (2 * i + t < tiles_here) {
            copy_scales(sfa + 4 * t, sfa0 + static_cast<uint64_t>(t * (kTileBytes >> 4)));
            copy_scales(sfx + 4 * t, sfx0 + static_cast<uint64_t>(t * (kTileBytes >> 4)));
#pragma unroll
            for (int j = 0; j < 2; ++j)
              mma_mxf4(tmem, a0 + 4 * t + 2 * j, b0 + 4 * t + 2 * j, mxf4_idesc(128, NB, j), sfa + 4 * t, sfx + 4 * t, (i | t | j) ? 1u : 0u);
          }
        }
        mma_commit(smem_u32(&hdr->empty[stage]));
        if (i == n_steps - 1) mma_commit(smem_u32(&hdr->done));
      }
      __syncwarp();
      if (++stage == p.stages) { stage = 0; phase ^= 1u; }
    }
  } else if (warp == 1) {       // the ring's later rounds
    int stage = 0;
    uint32_t phase = 0;
    for (; fetched < n_steps; ++fetched) {
      if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&hdr->empty[stage]), phase, &hdr->abort_flag, 0x4300u | stage))) { ok = false; break; }
      if (elect_one()) load_step(fetched, stage);
      __syncwarp();
      if (++stage == p.stages) { stage = 0; phase ^= 1u; }
    }
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
  __syncwarp();             // the cluster's barrier wants whole warps
  if (slices > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  if (warp == 1 && hdr->abort_flag != 0u) {   // someone gave up: a bounded wait for the last copies of every stage
    uint32_t left = kSpinLimit;
    for (int j = fetched - p.stages < 0 ? 0 : fetched - p.stages; j < fetched; ++j)
      while (left != 0u && !mbar_try_wait(smem_u32(&hdr->full[j % p.stages]), static_cast<uint32_t>(j / p.stages) & 1u)) --left;
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
    store_from_float(p.out.y, p.out.dtype, o,
                     p.out.dtype == DIMQ_F32 ? activate_any<true>(s, res, p.out.epilogue) : activate_any<false>(s, res, p.out.epilogue));
  }
  __syncwarp();
  if (slices > 1) {         // no block leaves while a peer may read its sums
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, columns_of(p.stages));
  }
}

template <int NB, typename T>
int launch_small(const CUtensorMap& codes, SmallParams p, bool vec, int64_t row_blocks, cudaStream_t st) {
  const size_t fixed = 1024 + p.room * (NB * 128 + 1024) + NB * 512 + sizeof(SmallHeader) + 64;
  // a ring as deep as leaves room for the blocks of this grid side by side (three to an SM at most)
  const int64_t blocks = row_blocks * p.slices, per_sm = blocks <= kNumSMs ? 1 : blocks <= 2 * kNumSMs ? 2 : 3;
  const int64_t free = static_cast<int64_t>(kSmemMax / per_sm) - 1024 - static_cast<int64_t>(fixed);
  p.stages = static_cast<int>(free / static_cast<int64_t>(kWeightBytes));
  if (p.stages > kMostStages) p.stages = kMostStages;
  if (p.stages > p.room) p.stages = p.room;
  if (p.stages < 2) p.stages = p.room < 2 ? 1 : 2;
  size_t smem = fixed + p.stages * kWeightBytes;
  const size_t least = columns_of(p.stages) / 64 * kBytesPer64Columns;
  if (smem < least) smem = least;
  auto kern = vec ? mx_small_kernel<NB, T, true> : mx_small_kernel<NB, T, false>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemMax));
  if (e != cudaSuccess) return static_cast<int>(e);
  e = launch_dependent(kern, static_cast<unsigned>(blocks), kThreads, smem, st, p.slices, codes, p);
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
}

template <typename T>
int small_as(const CUtensorMap& codes, const SmallParams& p, bool vec, int64_t row_blocks, cudaStream_t st) {
  if (p.out.rows <= 8) return launch_small<8, T>(codes, p, vec, row_blocks, st);
  if (p.out.rows <= 16) return launch_small<16, T>(codes, p, vec, row_blocks, st);
  return launch_small<32, T>(codes, p, vec, row_blocks, st);
}

}  // namespace

// Blocks of a cluster: as many as let the grid run side by side, three blocks to an SM
static int slices_of(int64_t row_blocks, int steps) {
  int slices = 1;
  while (slices < kMostSlices && 2 * slices <= steps &&
         (row_blocks * slices * 2 <= 3 * kNumSMs || (steps + slices - 1) / slices > kMostSteps))
    slices *= 2;
  return slices;
}

// Up to 16 rows always; up to 32 where a block's slice of x is short (1024 k): every block quantises its slice, so long
// ones cost more than a second launch (32 x 4096 -> 4096 8.3 us against 12.4, 32 x 8192 -> 8192 20.4 against 17.3).
bool mx_small_takes(int64_t M, int64_t N, int64_t K) {
  if (M > 32) return false;
  const int64_t steps = (mx::block_tiles(K) + 1) / 2, row_blocks = mx::row_tiles(N);
  if (steps > kMostSteps * kMostSlices || row_blocks > 0x7FFFFFFF / kMostSlices) return false;
  const int slices = slices_of(row_blocks, static_cast<int>(steps));
  return M <= 16 || (steps + slices - 1) / slices <= 4;
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
  const int slices = slices_of(row_blocks, p.steps);
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
