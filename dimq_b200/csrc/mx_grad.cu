// The gradients of the microscaled linear layer, straight through its rounding: dx = dy w^ and dw = dy^T x~.
//
// Both reduce over the slow axis of the coded operand (w^ [N][K] over n, x~ [M][K] over m), along which the block scales
// change, so the scales cannot be left to the block-scaled tensor cores.  A coded value is exact in bf16 (at most eight
// significant bits, bf16 has fp32's range), so the coded matrix is decoded once to scratch and multiplied by dy on the
// 16-bit tensor cores, fp32 sums.  Nothing is transposed: TMA brings boxes of 64 columns (the decoded matrix is written
// in panels of 64 columns, so that one copy brings all of a tile's), and the operand descriptors say that the columns are contiguous ("MN major") - w^ and x~ always, dy for dw.
//
// dy enters exactly: bf16 as it is, fp16 and fp32 as the sum of two or three bf16 terms, each the leading eight bits of
// what the ones before left (24 bits in all; an infinity or a NaN is its own first term).  bf16 has no bits under 2^-133, so an
// fp32 value loses what it has there: nothing above 2^-110, under 2.5e-7 of one of 2^-112, 6e-5 of 2^-120, 4e-3 of 2^-126.  The terms are passes over the
// same reduction, smallest first.
//
// The tensor cores cut their sums to fp32 instead of rounding them: the error grows with the number of steps.  Where the
// result is fp32 it is therefore added up in registers, 512 values of the reduction at a time.  A 16-bit result has room for
// some of that error: it is added up so where one accumulator would take more than 16384 (fp16) or 131072 (bf16) values of
// the reduction (long_steps).
//
// Tile: 128 rows x BN columns of the result, ring stages of 64 of the reduction, two accumulators in tensor memory.
// Warps 0-2 fetch, taking the stages in turn, warp 3 issues the MMAs, warps 4-11 are the epilogue, two to a lane quarter.
#include "mx_tile.cuh"

namespace dimq {
int mx_decode_panels(const void* codes, const uint8_t* scales, int format, int64_t rows, int64_t cols, void* out, cudaStream_t st);

namespace {

using namespace mx;

constexpr int kProducers = 3;
constexpr int kThreads = (kProducers + 1 + kEpiWarps) * 32;
constexpr int kMaxStages = 8;
constexpr int kDepth = 64;                       // reduction per stage
constexpr uint32_t kABytes = 128 * kDepth * 2;
constexpr int kSegStages = 8;

struct GradMaps {
  CUtensorMap a, b, y;
};

struct GradParams {
  Out out;
  int depth_blocks;        // 64-blocks of the reduction, per term
  int terms;
  int stages, n_tiles, m_tiles;
  int slices;              // parts of the reduction; more than one: fp32 partial results, [slice][rows][cols] at out.y
  int a_cols;              // dy's rows are the reduction (dw): its boxes are 64 columns x 64 rows
};

struct GradHeader {
  uint64_t full[kMaxStages], empty[kMaxStages], d_full[2], d_empty[2];
  uint32_t tmem_base, drained[2];
  volatile uint32_t abort_flag;
  uint32_t filled[kMaxStages];                   // how often each stage was
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* tmap, uint32_t bar, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const void* tmap, uint32_t bar, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void load_box(uint32_t dst, const void* tmap, uint32_t bar, int c0, int c1, int c2) {
  if (PAIR) tma_load_3d_pair(dst, tmap, bar, c0, c1, c2);
  else tma_load_3d(dst, tmap, bar, c0, c1, c2);
}
template <bool PAIR>
__device__ __forceinline__ void mma_bf16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// Columns contiguous: pieces of 64 columns x 8 rows of the reduction (1024 bytes, 128-byte swizzle), the next eight rows
// 1024 bytes on, the next 64 columns a whole box (64 rows) on.
__device__ __forceinline__ uint64_t columns_desc(uint32_t smem) {
  return static_cast<uint64_t>((smem & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(kDepth * 128 >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr) : "memory");
}

struct Unit {              // a block's piece of work: a part of the reduction of one tile
  int tile, slice, first, end;
};
__device__ __forceinline__ Unit unit_of(int u, int steps, const GradParams& p) {
  Unit w;
  w.tile = u / p.slices;
  w.slice = u - w.tile * p.slices;
  w.first = static_cast<int>(static_cast<int64_t>(steps) * w.slice / p.slices);
  w.end = static_cast<int>(static_cast<int64_t>(steps) * (w.slice + 1) / p.slices);
  return w;
}

// SEG: long sums, added up in registers.  PAIR: two blocks share a tile of 256 rows (BN = 256).
template <int BN, int ES, bool SEG, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
mx_grad_kernel(const __grid_constant__ GradMaps maps, const GradParams p) {
  constexpr int kCols = PAIR ? BN / 2 : BN;      // columns of the tile that this block holds
  constexpr uint32_t kStageBytes = kABytes + kCols * kDepth * 2;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t n_st = static_cast<uint32_t>(p.stages);
  GradHeader* hdr = reinterpret_cast<GradHeader*>(smem + n_st * kStageBytes);
  unsigned char* staging = reinterpret_cast<unsigned char*>(hdr) + kHeaderBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int all_steps = p.depth_blocks * p.terms, units = p.n_tiles * p.m_tiles * p.slices;
  const int rank = PAIR ? static_cast<int>(cluster_rank()) : 0;
  const int unit0 = PAIR ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int unit_step = PAIR ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) { mbar_init(smem_u32(&hdr->full[s]), 1); mbar_init(smem_u32(&hdr->empty[s]), 1); hdr->filled[s] = 0u; }
    for (int s = 0; s < 2; ++s) { mbar_init(smem_u32(&hdr->d_full[s]), 1); mbar_init(smem_u32(&hdr->d_empty[s]), PAIR ? 2 : 1); }
    hdr->abort_flag = 0u;
    hdr->drained[0] = hdr->drained[1] = 0u;
    fence_barrier_init();
    prefetch_tensormap(&maps.a);
    prefetch_tensormap(&maps.b);
    if (p.out.tma) prefetch_tensormap(&maps.y);
  }
  if (warp == kProducers) {
    if constexpr (PAIR) tmem_alloc_pair(smem_u32(&hdr->tmem_base), 512);
    else { tmem_alloc(smem_u32(&hdr->tmem_base), 512); tmem_relinquish(); }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if constexpr (PAIR) { cluster_arrive(); cluster_wait(); }   // the peer's barriers are there before anything signals them
  const uint32_t tmem = hdr->tmem_base;
  volatile uint32_t* abort_flag = &hdr->abort_flag;
  wait_for_inputs();

  if (warp < kProducers) {
    // no more producers than stages, as in the forward product
    const uint32_t turns = n_st < kProducers ? n_st : kProducers;
    uint32_t stage = 0, round = 0, turn = 0;
    bool ok = true;
    for (int u = unit0; u < units && ok; u += unit_step) {
      const Unit w = unit_of(u, all_steps, p);
      const int n_blk = w.tile % p.n_tiles, m_blk = (PAIR ? 2 : 1) * (w.tile / p.n_tiles) + rank;
      int term = p.terms - 1 - w.first / p.depth_blocks, kb = w.first % p.depth_blocks;   // smallest terms first
      for (int s = w.first; s < w.end; ++s) {
        if (turn == static_cast<uint32_t>(warp)) {
          if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&hdr->empty[stage]), (round & 1u) ^ 1u, abort_flag, 0x3100u | stage))) { ok = false; break; }
          const uint32_t full = smem_u32(&hdr->full[stage]), dst = smem_u32(smem + stage * kStageBytes);
          if (elect_one()) {     // a pair counts both blocks' bytes in the first one's barrier
            hdr->filled[stage] = round + 1u;
            if (rank == 0) mbar_arrive_expect_tx(full, (PAIR ? 2 : 1) * kStageBytes);
            const uint32_t bar = PAIR ? map_to_cta(full, 0) : full;
            if (p.a_cols) {
              load_box<PAIR>(dst, &maps.a, bar, m_blk * 128, kb * kDepth, term);
              load_box<PAIR>(dst + kABytes / 2, &maps.a, bar, m_blk * 128 + 64, kb * kDepth, term);
            } else {
              load_box<PAIR>(dst, &maps.a, bar, kb * kDepth, m_blk * 128, term);
            }
            load_box<PAIR>(dst + kABytes, &maps.b, bar, 0, kb * kDepth, n_blk * (BN / 64) + rank * (kCols / 64));
          }
          __syncwarp();
        }
        if (++turn == turns) turn = 0;
        if (++stage == n_st) { stage = 0; ++round; }
        if (++kb == p.depth_blocks) { kb = 0; --term; }
      }
    }
    __syncwarp();
  } else if (warp == kProducers) {
    uint32_t stage = 0, phase = 0, buf = 0, bph = 0;
    bool ok = rank == 0;      // the first block of a pair issues for both
    const uint32_t idesc = make_idesc_f16(1, 1, PAIR ? 256 : 128, BN) | (p.a_cols ? 1u << 15 : 0u) | (1u << 16);
    const uint64_t a_step = p.a_cols ? 2048 >> 4 : 32 >> 4;   // 16 of the reduction
    for (int u = unit0; u < units && ok; u += unit_step) {
      const Unit w = unit_of(u, all_steps, p);
      for (int seg0 = w.first; seg0 < w.end && ok; seg0 += SEG ? kSegStages : all_steps) {
        const int seg1 = SEG && seg0 + kSegStages < w.end ? seg0 + kSegStages : w.end;
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&hdr->d_empty[buf]), bph ^ 1u, abort_flag, 0x3200u | buf))) { ok = false; break; }
        tc_fence_after();
        const uint32_t d = tmem + buf * 256;
        for (int s = seg0; s < seg1; ++s) {
          if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&hdr->full[stage]), phase, abort_flag, 0x3300u | stage))) { ok = false; break; }
          tc_fence_after();
          const uint32_t at = smem_u32(smem + stage * kStageBytes);
          const uint64_t a0 = p.a_cols ? columns_desc(at) : make_smem_desc_sw128(at), b0 = columns_desc(at + kABytes);
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < kDepth / 16; ++j)
              mma_bf16<PAIR>(d, a0 + a_step * j, b0 + static_cast<uint64_t>((2048 >> 4) * j), idesc, (s > seg0 || j) ? 1u : 0u);
            commit<PAIR>(smem_u32(&hdr->empty[stage]));
          }
          __syncwarp();
          if (++stage == n_st) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        if (elect_one()) commit<PAIR>(smem_u32(&hdr->d_full[buf]));
        __syncwarp();
        if (++buf == 2) { buf = 0; bph ^= 1u; }
      }
    }
  } else {
    const int ew = warp - kProducers - 1;
    const int quarter = warp & 3, sub = ew >> 2;
    unsigned char* stage = staging + ew * kStagingBytes;
    constexpr int kMine = BN / 64;
    uint32_t buf = 0, bph = 0, piece = 0;
    bool ok = true;
    Out out = p.out;
    for (int u = unit0; u < units && ok; u += unit_step) {
      const Unit w = unit_of(u, all_steps, p);
      const int64_t n_first = static_cast<int64_t>(w.tile % p.n_tiles) * BN, tile_row0 = (static_cast<int64_t>(PAIR ? 2 : 1) * (w.tile / p.n_tiles) + rank) * 128 + quarter * 32;
      // partial results lie one under the other: a slice's rows start at slice * rows.  Only whole pieces of 32 rows go
      // through the map; a piece that ends in the next slice's rows is stored plainly.
      const int64_t row_off = static_cast<int64_t>(w.slice) * p.out.rows, row0 = tile_row0 + row_off;
      out.rows = p.out.rows + row_off;
      out.tma = p.out.tma && (p.slices == 1 || tile_row0 + 32 <= p.out.rows);
      const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
      float sum[SEG ? kMine : 1][32];
      for (int seg0 = w.first; seg0 < w.end; seg0 += SEG ? kSegStages : all_steps) {
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&hdr->d_full[buf]), bph, abort_flag, 0x3500u | buf))) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          const uint32_t col = tmem + lanes + buf * 256 + (sub + 2 * i) * 32;
          if constexpr (SEG) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t r[16];
              tmem_ld16(col + 16 * h, r);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) sum[i][16 * h + j] = (seg0 == w.first ? 0.0f : sum[i][16 * h + j]) + __uint_as_float(r[j]);
            }
          } else {
            uint32_t r[32];
            tmem_ld32(col, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[0][j] = __uint_as_float(r[j]);
          }
          if (i == kMine - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) hand_back<PAIR>(&hdr->drained[buf], smem_u32(&hdr->d_empty[buf]));
          }
          __syncwarp();
          if constexpr (!SEG) {
            const int64_t n0 = n_first + (sub + 2 * i) * 32;
            if (row0 < out.rows && n0 < out.cols) put_chunk<ES, false>(sum[0], out, &maps.y, stage, piece, nullptr, row0, n0, lane);
          }
        }
        if (++buf == 2) { buf = 0; bph ^= 1u; }
      }
      if (!ok) break;
      if constexpr (SEG) {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          const int64_t n0 = n_first + (sub + 2 * i) * 32;
          if (row0 < out.rows && n0 < out.cols) put_chunk<ES, false>(sum[i], out, &maps.y, stage, piece, nullptr, row0, n0, lane);
        }
      }
    }
    __syncwarp();
    if (elect_one()) tma_store_wait_all();
    __syncwarp();
  }

  tc_fence_before();
  leave_together<PAIR>(abort_flag, hdr->full, hdr->filled, n_st, rank);
  if (warp == kProducers) {
    tc_fence_after();
    if constexpr (PAIR) tmem_dealloc_pair(tmem, 512);
    else tmem_dealloc(tmem, 512);
  }
}

// dy [rows][cols] -> TERMS bf16 matrices [rows][pitch] whose sum it is; zeros behind the last column
template <typename T, int TERMS>
__global__ void __launch_bounds__(256)
mx_terms_kernel(const T* __restrict__ dy, int64_t rows, int64_t cols, int64_t pitch, uint16_t* __restrict__ out) {
  const int64_t per_row = pitch / 8;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; u < rows * per_row; u += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = u / per_row, c = (u - row * per_row) * 8;
    uint32_t w[TERMS][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = c + i < cols ? to_float<T>(dy[row * cols + c + i]) : 0.0f;
#pragma unroll
      for (int t = 0; t < TERMS; ++t) {
        uint32_t h = __float_as_uint(v) >> 16;       // cut, not rounded: a large value stays finite
        if (v != v) h = 0x7FFFu;
        const float f = __uint_as_float(h << 16);
        v = (h & 0x7F80u) == 0x7F80u ? 0.0f : v - f;
        if (i & 1) w[t][i >> 1] |= h << 16;
        else w[t][i >> 1] = h;
      }
    }
#pragma unroll
    for (int t = 0; t < TERMS; ++t)
      *reinterpret_cast<uint4*>(out + (t * rows + row) * pitch + c) = make_uint4(w[t][0], w[t][1], w[t][2], w[t][3]);
  }
}

// sums of the slices, in order
template <typename T>
__global__ void __launch_bounds__(256)
mx_add_slices_kernel(const float* __restrict__ partial, int slices, int64_t n, T* __restrict__ out) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  if (n % 4 == 0) {
    float4 s = *reinterpret_cast<const float4*>(partial + i);
    for (int r = 1; r < slices; ++r) {
      const float4 v = *reinterpret_cast<const float4*>(partial + r * n + i);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    out[i] = from_float<T>(s.x); out[i + 1] = from_float<T>(s.y); out[i + 2] = from_float<T>(s.z); out[i + 3] = from_float<T>(s.w);
  } else {
    for (int64_t j = i; j < i + 4 && j < n; ++j) {
      float s = partial[j];
      for (int r = 1; r < slices; ++r) s += partial[r * n + j];
      out[j] = from_float<T>(s);
    }
  }
}

// Column sums: a block takes 256 columns of a run of rows (the grid is one dimension: run, then columns), its eight warps the
// rows in turn; the runs' sums are added by a second kernel, in order.  VEC: rows of whole 16-byte pieces, a lane has eight
// neighbours; else columns 32 apart.
constexpr int kSumRows = 256;
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
mx_column_sum_kernel(const T* __restrict__ dy, int64_t rows, int64_t cols, unsigned col_tiles, float* __restrict__ partial,
                     void* __restrict__ out, int out_dtype) {
  __shared__ float part[8][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned run = blockIdx.x / col_tiles;
  const int64_t c0 = static_cast<int64_t>(blockIdx.x - run * col_tiles) * 256;
  const int64_t r0 = static_cast<int64_t>(run) * kSumRows, r1 = r0 + kSumRows < rows ? r0 + kSumRows : rows;
  float s[8] = {};
#pragma unroll 4
  for (int64_t r = r0 + warp; r < r1; r += 8) {
    if (VEC) {
      const Eight<T> e = load_pieces<T>(dy + r * cols, c0 + 8 * lane, cols);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = pair_of(e, i);
        s[2 * i] += v.x;
        s[2 * i + 1] += v.y;
      }
    } else {
      T v[8];
      load_neighbours<T>(dy + r * cols, c0, cols, lane, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += to_float<T>(v[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) part[warp][VEC ? 8 * lane + i : 32 * i + lane] = s[i];
  __syncthreads();
  const int64_t j = c0 + threadIdx.x;
  if (j >= cols) return;
  float t = part[0][threadIdx.x];
  for (int i = 1; i < 8; ++i) t += part[i][threadIdx.x];
  if (rows > kSumRows) partial[run * cols + j] = t;
  else store_from_float(out, out_dtype, j, t);
}
__global__ void __launch_bounds__(128)
mx_column_sum_finish_kernel(const float* __restrict__ partial, int64_t runs, int64_t cols, void* __restrict__ out, int out_dtype) {
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x;
  if (j >= cols) return;
  float s = 0.0f;
#pragma unroll 8
  for (int64_t r = 0; r < runs; ++r) s += partial[r * cols + j];
  store_from_float(out, out_dtype, j, s);
}

template <typename T>
int column_sum(const void* dy, int64_t M, int64_t N, float* partial, void* db, int db_dtype, cudaStream_t st) {
  const int64_t runs = (M + kSumRows - 1) / kSumRows, gx = (N + 255) / 256;
  if (gx > 0x7FFFFFFF / runs) return DIMQ_ERR_TOO_LARGE;   // 1.4e14 values
  const unsigned cols = static_cast<unsigned>(gx), grid = cols * static_cast<unsigned>(runs);
  const T* in = static_cast<const T*>(dy);
  if ((N * static_cast<int64_t>(sizeof(T))) % 16 == 0) mx_column_sum_kernel<T, true><<<grid, 256, 0, st>>>(in, M, N, cols, partial, db, db_dtype);
  else mx_column_sum_kernel<T, false><<<grid, 256, 0, st>>>(in, M, N, cols, partial, db, db_dtype);
  const int rc = launch_status();
  if (rc != DIMQ_OK || runs == 1) return rc;
  mx_column_sum_finish_kernel<<<static_cast<unsigned>((N + 127) / 128), 128, 0, st>>>(partial, runs, N, db, db_dtype);
  return launch_status();
}

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

int terms_of(int dtype) { return dtype == DIMQ_BF16 ? 1 : dtype == DIMQ_F16 ? 2 : 3; }
bool as_it_is(int dtype, int64_t cols) { return dtype == DIMQ_BF16 && cols % 8 == 0; }
int64_t decoded_bytes(int64_t rows, int64_t K) { return up(rows * up(K, 64) * 2, 256); }
int64_t terms_bytes(int dtype, int64_t M, int64_t N) { return as_it_is(dtype, N) ? 0 : up(terms_of(dtype) * M * up(N, 8) * 2, 256); }
int64_t partial_bytes(int64_t M, int64_t N) { return M > kSumRows ? up((M + kSumRows - 1) / kSumRows * N * 4, 256) : 0; }

// dy as the tensor cores take it: itself, or its terms in scratch
int split_terms(const void* dy, int dtype, int64_t M, int64_t N, void* scratch, const void** a, int64_t* pitch, cudaStream_t st) {
  *a = dy;
  *pitch = N;
  if (as_it_is(dtype, N)) return DIMQ_OK;
  *a = scratch;
  *pitch = up(N, 8);
  const int64_t units = M * (*pitch / 8), blocks = (units + 255) / 256;
  const unsigned grid = static_cast<unsigned>(blocks < kNumSMs * 16 ? blocks : kNumSMs * 16);
  uint16_t* out = static_cast<uint16_t*>(scratch);
  if (dtype == DIMQ_F32) mx_terms_kernel<float, 3><<<grid, 256, 0, st>>>(static_cast<const float*>(dy), M, N, *pitch, out);
  else if (dtype == DIMQ_F16) mx_terms_kernel<__half, 2><<<grid, 256, 0, st>>>(static_cast<const __half*>(dy), M, N, *pitch, out);
  else mx_terms_kernel<__nv_bfloat16, 1><<<grid, 256, 0, st>>>(static_cast<const __nv_bfloat16*>(dy), M, N, *pitch, out);
  return launch_status();
}

template <int BN, int ES, bool SEG, bool PAIR>
int launch_grad(GradMaps& maps, GradParams& p, cudaStream_t st) {
  constexpr size_t kRing = kABytes + (PAIR ? BN / 2 : BN) * kDepth * 2;
  const size_t fixed = 1024 + kHeaderBytes + kEpiWarps * kStagingBytes;
  p.stages = static_cast<int>((kSmemMax - fixed) / kRing);
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  auto kern = mx_grad_kernel<BN, ES, SEG, PAIR>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemMax));
  if (e != cudaSuccess) return static_cast<int>(e);
  const int64_t units = static_cast<int64_t>(p.m_tiles) * p.n_tiles * p.slices, most = PAIR ? kNumSMs / 2 : kNumSMs;
  const unsigned grid = static_cast<unsigned>((units < most ? units : most) * (PAIR ? 2 : 1));
  e = launch_dependent(kern, grid, kThreads, fixed + p.stages * kRing, st, PAIR ? 2 : 1, maps, p);
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
}

// How a product [R][K] over `depth` (times terms) is cut: tile width and slices of the reduction, by what waves of units
// cost (cycles of a 64-step of each width) and, where it is sliced, what the partial results cost to write and to add
// (about 3 KB a cycle over the whole chip, and a launch).  The weight gradient of 25216 tokens, 2304 x 768: 54 tiles of 256
// columns took 170 us whole, 106 in slices.
struct GradPlan {
  int bn, slices;     // bn 512: pairs of blocks, 256 x 256
};
GradPlan plan_of(int64_t R, int64_t K, int64_t depth, int terms) {
  const int form[4] = {512, 256, 128, 64};
  const double cost[4] = {650.0, 750.0, 520.0, 430.0};
  const int64_t steps = (depth + kDepth - 1) / kDepth * terms;
  GradPlan best = {512, 1};
  double least = -1.0;
  for (int i = 0; i < 4; ++i) {
    const int64_t width = form[i] > 256 ? 256 : form[i], side_by_side = form[i] > 256 ? kNumSMs / 2 : kNumSMs;
    const int64_t tiles = (form[i] > 256 ? (row_tiles(R) + 1) / 2 : row_tiles(R)) * ((K + width - 1) / width);
    for (int s = 1; s <= 16 && (s == 1 || (s * kSegStages <= steps && tiles * (s - 1) < side_by_side)); ++s) {
      const double waves = static_cast<double>((tiles * s + side_by_side - 1) / side_by_side);
      double c = waves * (static_cast<double>((steps + s - 1) / s) * cost[i] + 2000.0);
      if (s > 1) c += 6000.0 + static_cast<double>(R) * K * 8 * s / 3000.0;
      if (least < 0.0 || c < least) { least = c; best = {form[i], s}; }
    }
  }
  return best;
}
int64_t slices_bytes(int64_t R, int64_t K, int64_t depth, int terms) {
  const int s = plan_of(R, K, depth, terms).slices;
  return s > 1 ? up(R * K * 4 * s, 256) : 0;
}

// Steps (of 64 values, of one term: the smaller terms' sums are small) after which an accumulator's cuts would count in a
// 16-bit result.  Values of one sign lose 8e-8 of the sum per 16 values: 6.5e-4 of an fp16 weight gradient over a million
// rows (in 16 slices), more than half a step of fp16 (4.9e-4).  These limits keep that below a sixth of half a step.
int64_t long_steps(int dtype) { return dtype == DIMQ_F16 ? 256 : 2048; }

// out [R][K] = A * decoded, A = dy (reduction over its columns) or dy^T (over its rows, a_cols); `depth` values reduced
int grad_product(const void* dy, int64_t M, int64_t N, int64_t pitch, int terms, bool a_cols, const void* decoded, int64_t depth, int64_t K,
                 Out out, void* partial, cudaStream_t st) {
  GradMaps maps;
  GradParams p = {};
  const GradPlan plan = plan_of(out.rows, K, depth, terms);
  const bool pair = plan.bn > 256;
  const int bn = pair ? 256 : plan.bn;
  const Out result = out;
  if (plan.slices > 1) {
    out.y = partial;
    out.dtype = DIMQ_F32;
  }
  out.tma = out_by_map(out);
  p.out = out;
  p.terms = terms;
  p.slices = plan.slices;
  p.a_cols = a_cols;
  p.depth_blocks = static_cast<int>((depth + kDepth - 1) / kDepth);
  const int64_t n_tiles = (K + bn - 1) / bn, m_tiles = pair ? (row_tiles(out.rows) + 1) / 2 : row_tiles(out.rows);
  if (n_tiles * m_tiles * plan.slices > 0x7FFFFFFF - kNumSMs || static_cast<int64_t>(p.depth_blocks) * terms > 0x7FFFFFFF - 64 ||
      out.rows * plan.slices > 0x7FFFFF00)
    return DIMQ_ERR_TOO_LARGE;
  p.n_tiles = static_cast<int>(n_tiles);
  p.m_tiles = static_cast<int>(m_tiles);
  const CUtensorMapDataType bf16 = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const cuuint64_t adims[3] = {static_cast<cuuint64_t>(N), static_cast<cuuint64_t>(M), static_cast<cuuint64_t>(terms)};
  const cuuint64_t astr[2] = {static_cast<cuuint64_t>(pitch) * 2, static_cast<cuuint64_t>(pitch) * 2 * static_cast<cuuint64_t>(M)};
  const cuuint32_t abox[3] = {64, a_cols ? 64u : 128u, 1};
  const cuuint64_t bdims[3] = {64, static_cast<cuuint64_t>(depth), static_cast<cuuint64_t>(up(K, 64) / 64)};
  const cuuint64_t bstr[2] = {128, static_cast<cuuint64_t>(depth) * 128};
  const cuuint32_t bbox[3] = {64, kDepth, static_cast<cuuint32_t>((pair ? bn / 2 : bn) / 64)};
  Out rows_of_all = out;
  rows_of_all.rows *= plan.slices;
  if (!encode_map(&maps.a, bf16, 3, dy, adims, astr, abox, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode_map(&maps.b, bf16, 3, decoded, bdims, bstr, bbox, CU_TENSOR_MAP_SWIZZLE_128B) ||
      (out.tma && !encode_out(&maps.y, rows_of_all)))
    return DIMQ_ERR_DRIVER;
  const bool wide = result.dtype == DIMQ_F32;
  const int64_t steps = static_cast<int64_t>(p.depth_blocks) * terms, share = (steps + plan.slices - 1) / plan.slices;
  const bool seg = wide ? steps > kSegStages * plan.slices
                        : (share < p.depth_blocks ? share : p.depth_blocks) > long_steps(result.dtype);
  int rc;
#define DIMQ_MX_GRAD(ES, SEG)                                          \
  rc = pair ? launch_grad<256, ES, SEG, true>(maps, p, st)             \
       : bn == 256 ? launch_grad<256, ES, SEG, false>(maps, p, st)     \
       : bn == 128 ? launch_grad<128, ES, SEG, false>(maps, p, st) : launch_grad<64, ES, SEG, false>(maps, p, st)
  if (seg && out.dtype == DIMQ_F32) { DIMQ_MX_GRAD(4, true); }
  else if (seg) { DIMQ_MX_GRAD(2, true); }
  else if (out.dtype == DIMQ_F32) { DIMQ_MX_GRAD(4, false); }
  else { DIMQ_MX_GRAD(2, false); }
#undef DIMQ_MX_GRAD
  if (rc != DIMQ_OK || plan.slices == 1) return rc;
  const int64_t n = out.rows * out.cols, blocks = (n + 1023) / 1024;
  if (blocks > 0x7FFFFFFF) return DIMQ_ERR_TOO_LARGE;
  const unsigned grid = static_cast<unsigned>(blocks);
  const float* from = static_cast<const float*>(partial);
  if (wide) mx_add_slices_kernel<float><<<grid, 256, 0, st>>>(from, plan.slices, n, static_cast<float*>(result.y));
  else if (result.dtype == DIMQ_F16) mx_add_slices_kernel<__half><<<grid, 256, 0, st>>>(from, plan.slices, n, static_cast<__half*>(result.y));
  else mx_add_slices_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(from, plan.slices, n, static_cast<__nv_bfloat16*>(result.y));
  return launch_status();
}

int check_sizes(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N <= 0 || K <= 0) return DIMQ_ERR_BAD_SIZE;
  if (M > 0x7FFFFF00 || N > 0x7FFFFF00 || K > 0x7FFFFF00) return DIMQ_ERR_TOO_LARGE;
  return DIMQ_OK;
}

int64_t grad_bytes(int dtype, int64_t M, int64_t N, int64_t K) {
  const int terms = terms_of(dtype);
  const int64_t in = slices_bytes(M, K, N, terms), weight = slices_bytes(N, K, M, terms), sums = partial_bytes(M, N);
  const int64_t most = in > weight ? in : weight;
  return decoded_bytes(M > N ? M : N, K) + terms_bytes(dtype, M, N) + (most > sums ? most : sums);
}

int clear(void* p, int dtype, int64_t n, cudaStream_t st) {   // a sum over no rows
  const cudaError_t e = cudaMemsetAsync(p, 0, static_cast<size_t>(n) * dtype_size(dtype), st);
  return e == cudaSuccess ? DIMQ_OK : static_cast<int>(e);
}

}  // namespace

int read_mx_grad_status(uint32_t* status) { return tc::read_and_clear_device_status(status); }

}  // namespace dimq

using namespace dimq;

extern "C" int dimq_mx_grad_workspace_bytes(int dy_dtype, int64_t M, int64_t N, int64_t K, int64_t* bytes) {
  if (bytes == nullptr) return DIMQ_ERR_NULL_POINTER;
  *bytes = 0;
  if (!valid_dtype(dy_dtype)) return DIMQ_ERR_BAD_DTYPE;
  const int rc = check_sizes(M, N, K);
  if (rc != DIMQ_OK) return rc;
  *bytes = grad_bytes(dy_dtype, M, N, K);
  return DIMQ_OK;
}

extern "C" int dimq_mx_grad_launches(int dy_dtype, int64_t M, int64_t N, int64_t K, int dx, int dw, int db, int* kernels) {
  if (kernels == nullptr) return DIMQ_ERR_NULL_POINTER;
  *kernels = 0;
  if (!valid_dtype(dy_dtype)) return DIMQ_ERR_BAD_DTYPE;
  const int rc = check_sizes(M, N, K);
  if (rc != DIMQ_OK || M == 0) return rc;
  const int terms = terms_of(dy_dtype);
  if (db) *kernels += 1 + (M > kSumRows);                                             // runs, their sum
  if ((dx || dw) && !as_it_is(dy_dtype, N)) *kernels += 1;                            // terms
  if (dx) *kernels += 2 + (plan_of(M, K, N, terms).slices > 1);                       // decode, product, sum of slices
  if (dw) *kernels += 2 + (plan_of(N, K, M, terms).slices > 1);
  return DIMQ_OK;
}

// dx (null: not wanted) from w, dw (null) from x, db (null); dy's terms are made once
static int grads(const void* dy, int dy_dtype, const uint8_t* w_codes, const uint8_t* w_scales, const void* x_codes,
                 const uint8_t* x_scales, int format, void* dx, int dx_dtype, void* dw, int dw_dtype, void* db, int db_dtype, int64_t M,
                 int64_t N, int64_t K, void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_sizes(M, N, K);
  if (rc != DIMQ_OK) return rc;
  if (dw != nullptr && !mx::valid_format(format)) return DIMQ_ERR_BAD_BITS;
  if (!valid_dtype(dy_dtype) || (dx != nullptr && !valid_dtype(dx_dtype)) || (dw != nullptr && !valid_dtype(dw_dtype)) ||
      (db != nullptr && !valid_dtype(db_dtype)))
    return DIMQ_ERR_BAD_DTYPE;
  if (M > 0 && (dy == nullptr || (dx != nullptr && (w_codes == nullptr || w_scales == nullptr)) ||
                (dw != nullptr && (x_codes == nullptr || x_scales == nullptr))))
    return DIMQ_ERR_NULL_POINTER;
  if (!aligned(dy, 16) || !aligned(w_codes, 16) || !aligned(w_scales, 16) || !aligned(x_codes, 16) || !aligned(x_scales, 16) ||
      !aligned(workspace, 256))
    return DIMQ_ERR_ALIGNMENT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (M == 0) {
    if (dw != nullptr) rc = clear(dw, dw_dtype, N * K, st);
    if (rc == DIMQ_OK && db != nullptr) rc = clear(db, db_dtype, N, st);
    return rc;
  }
  if (workspace == nullptr || workspace_bytes < grad_bytes(dy_dtype, M, N, K)) return DIMQ_ERR_SCRATCH_TOO_SMALL;
  unsigned char* decoded = static_cast<unsigned char*>(workspace);
  unsigned char* split = decoded + decoded_bytes(M > N ? M : N, K);
  float* partial = reinterpret_cast<float*>(split + terms_bytes(dy_dtype, M, N));
  if (db != nullptr) {
    rc = dy_dtype == DIMQ_F32 ? column_sum<float>(dy, M, N, partial, db, db_dtype, st)
         : dy_dtype == DIMQ_F16 ? column_sum<__half>(dy, M, N, partial, db, db_dtype, st)
                                : column_sum<__nv_bfloat16>(dy, M, N, partial, db, db_dtype, st);
    if (rc != DIMQ_OK) return rc;
  }
  if (dx == nullptr && dw == nullptr) return DIMQ_OK;
  const void* a;
  int64_t pitch;
  const int terms = terms_of(dy_dtype);
  rc = split_terms(dy, dy_dtype, M, N, split, &a, &pitch, st);
  if (rc != DIMQ_OK) return rc;
  if (dx != nullptr) {
    rc = mx_decode_panels(w_codes, w_scales, DIMQ_MX_FP4, N, K, decoded, st);
    if (rc != DIMQ_OK) return rc;
    rc = grad_product(a, M, N, pitch, terms, false, decoded, N, K, {dx, nullptr, nullptr, M, K, 0, dx_dtype, DIMQ_EPI_NONE, 0}, partial, st);
    if (rc != DIMQ_OK) return rc;
  }
  if (dw != nullptr) {
    rc = mx_decode_panels(x_codes, x_scales, format, M, K, decoded, st);
    if (rc != DIMQ_OK) return rc;
    rc = grad_product(a, M, N, pitch, terms, true, decoded, M, K, {dw, nullptr, nullptr, N, K, 0, dw_dtype, DIMQ_EPI_NONE, 0}, partial, st);
  }
  return rc;
}

extern "C" int dimq_mx_grad_input(const void* dy, int dy_dtype, const uint8_t* w_codes, const uint8_t* w_scales, void* dx,
                                  int dx_dtype, int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  if (dx == nullptr && M > 0) return DIMQ_ERR_NULL_POINTER;
  return grads(dy, dy_dtype, w_codes, w_scales, nullptr, nullptr, 0, dx, dx_dtype, nullptr, 0, nullptr, 0, M, N, K, workspace,
               workspace_bytes, stream);
}

extern "C" int dimq_mx_grad_weight(const void* dy, int dy_dtype, const void* x_codes, const uint8_t* x_scales, int format, void* dw,
                                   int dw_dtype, void* db, int db_dtype, int64_t M, int64_t N, int64_t K, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  if (dw == nullptr && db == nullptr) return DIMQ_ERR_NULL_POINTER;
  return grads(dy, dy_dtype, nullptr, nullptr, x_codes, x_scales, format, nullptr, 0, dw, dw_dtype, db, db_dtype, M, N, K, workspace,
               workspace_bytes, stream);
}

extern "C" int dimq_mx_grads(const void* dy, int dy_dtype, const uint8_t* w_codes, const uint8_t* w_scales, const void* x_codes,
                             const uint8_t* x_scales, int format, void* dx, int dx_dtype, void* dw, int dw_dtype, void* db, int db_dtype,
                             int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes, void* stream) {
  if (dx == nullptr && dw == nullptr && db == nullptr) return DIMQ_ERR_NULL_POINTER;
  return grads(dy, dy_dtype, w_codes, w_scales, x_codes, x_scales, format, dx, dx_dtype, dw, dw_dtype, db, db_dtype, M, N, K, workspace,
               workspace_bytes, stream);
}
