// The microscaled 4-bit product y = x^ w^T on the block-scaled tensor cores.
//
// tcgen05.mma kind::mxf4 multiplies e2m1 codes as they are stored, 64 of them a step, and scales each block of 32 by the
// two operands' powers of two before it adds: products and scaling are exact, sums are fp32.  So nothing is decoded: TMA
// brings codes (rows of 128 bytes = 256 values, 128-byte swizzle) and the 512-byte scale tiles that the format keeps,
// tcgen05.cp moves a scale tile to tensor memory, and the accumulators go through bias, activation and residual to y.
// Products are multiples of a quarter of their blocks' scales and 64 of them take one step, so the cut to fp32 at each step
// often loses nothing: the sums of normal values, of mixed or one sign, are exact (K = 32768).  Where scales are spread, each
// step cuts up to 2^-23 of the sum, always towards zero (relative Frobenius norms at K = 8192 / 32768): scales over 2^+-4 on
// either side, mixed signs, 1.3e-7 / 7.9e-7; over 2^+-12, 2.6e-6 / 1.0e-5; over 2^+-6, all of one sign, 1.7e-6 / 8.0e-6.  An
// fp32 torch.matmul of the same values is off by 1.4e-7 / 4.5e-7, 6.3e-7 / 1.2e-6 and 5.5e-6 / 2.9e-5 (1300 x 2600).  Adding up
// parts of K in registers would bring these down; it took 58 us instead of 40 (2048 x 11008 -> 2048) and was left out.
//
// Large problems run on pairs of blocks (cta_group::2): 256 x 256 tiles, each block holding its 128 rows of x and half of
// the tile's rows of w, so that a step moves 32 KB of codes into each shared memory instead of 48.  The first block of a
// pair issues for both; the scales of w are in both tensor memories.
//
// Tile: 128 rows of x (one tensor-memory lane each) x BN rows of w.  A ring stage holds 256 k of both operands and their
// scales; its scale columns in tensor memory belong to the stage too, so the commit that frees the stage frees them.
// Warps 0-2 fetch (they take the stages in turn), warp 3 issues copies and MMAs, warps 4-11 are the epilogue: two to each
// quarter of the lanes, taking 32-column pieces in turn.  Persistent grid, one block per SM.
#include "mx_tile.cuh"

namespace dimq {
int mx_quantize(const void* x, int x_dtype, int64_t rows, int64_t cols, void* c4, uint8_t* s4, void* c8, uint8_t* s8,
                cudaStream_t st);
bool mx_small_takes(int64_t M, int64_t N, int64_t K);
int mx_small(const void* x, int x_dtype, const uint8_t* wc, const uint8_t* ws, const void* bias, int bias_dtype, const void* residual,
             void* y, int y_dtype, int64_t M, int64_t N, int64_t K, int epilogue, cudaStream_t st);

namespace {

using namespace mx;

constexpr int kProducers = 3;
constexpr int kThreads = (kProducers + 1 + kEpiWarps) * 32;
constexpr int kMaxStages = 8;
constexpr int kSfCol = 256;                      // first tensor-memory column of the scales
constexpr uint32_t kABytes = 128 * 128;
constexpr int kBiasBytes = kEpiWarps * 4 * 128;  // four pieces of 32 columns a warp

struct GemmMaps {
  CUtensorMap a, b, y, sfa, sfb;   // scales: pairs only
};

struct GemmParams {
  const uint8_t *sfa, *sfb;
  Out out;
  int k_tiles;             // scale tiles along k (128 values each)
  int row_tiles_b;         // scale tiles along n
  int stages, n_tiles, tiles;
};

struct GemmHeader {
  uint64_t full[kMaxStages], empty[kMaxStages], d_full[2], d_empty[2];
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
  uint32_t filled[kMaxStages];                   // how often each stage was
};

template <int BN, bool PAIR>
struct Shape {
  static constexpr int kRowTiles = BN > 128 ? BN / 128 : 1;               // scale tiles of w a stage holds per k tile
  static constexpr uint32_t kBBytes = (PAIR ? BN / 2 : BN) * 128;
  static constexpr uint32_t kStageBytes = kABytes + kBBytes + 1024 + kRowTiles * 1024;
  static constexpr int kSfCols = 8 + 8 * kRowTiles;                      // tensor-memory columns of a stage's scales
  static constexpr int kBufs = BN > 128 ? 1 : 2;                         // accumulators
  static constexpr int kMost = (512 - kSfCol) / kSfCols < kMaxStages ? (512 - kSfCol) / kSfCols : kMaxStages;
};

// PAIR: BN = 256.
template <int BN, int ES, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
mx_gemm_kernel(const __grid_constant__ GemmMaps maps, const GemmParams p) {
  using S = Shape<BN, PAIR>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t n_st = static_cast<uint32_t>(p.stages);
  GemmHeader* hdr = reinterpret_cast<GemmHeader*>(smem + n_st * S::kStageBytes);
  float* biases = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(hdr) + kHeaderBytes);
  unsigned char* staging = reinterpret_cast<unsigned char*>(biases) + kBiasBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int k_stages = (p.k_tiles + 1) / 2;
  const int rank = PAIR ? static_cast<int>(cluster_rank()) : 0;
  const int tile0 = PAIR ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int tile_step = PAIR ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) { mbar_init(smem_u32(&hdr->full[s]), 1); mbar_init(smem_u32(&hdr->empty[s]), 1); hdr->filled[s] = 0u; }
    for (int s = 0; s < 2; ++s) { mbar_init(smem_u32(&hdr->d_full[s]), 1); mbar_init(smem_u32(&hdr->d_empty[s]), PAIR ? 2 : 1); }
    hdr->abort_flag = 0u;
    fence_barrier_init();
    prefetch_tensormap(&maps.a);
    prefetch_tensormap(&maps.b);
    if (p.out.tma) prefetch_tensormap(&maps.y);
  }
  if (warp == kProducers) {
    if constexpr (PAIR) tmem_alloc_pair(smem_u32(&hdr->tmem_base), 512);   // the same columns in both
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
    // no more producers than stages: a warp's successive stages are at most one revolution apart, or the one bit of a
    // barrier's phase could not tell the round it waits for from the one before
    const uint32_t turns = n_st < kProducers ? n_st : kProducers;
    uint32_t stage = 0, round = 0, turn = 0;
    bool ok = true;
    for (int t = tile0; t < p.tiles && ok; t += tile_step) {
      const int n_blk = t % p.n_tiles, m_blk = (PAIR ? 2 : 1) * (t / p.n_tiles) + rank;
      for (int kb = 0; kb < k_stages; ++kb) {
        if (turn == static_cast<uint32_t>(warp)) {
          if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&hdr->empty[stage]), (round & 1u) ^ 1u, abort_flag, 0x2100u | stage))) { ok = false; break; }
          const uint32_t full = smem_u32(&hdr->full[stage]), dst = smem_u32(smem + stage * S::kStageBytes);
          const uint32_t sf = dst + kABytes + S::kBBytes;
          if constexpr (PAIR) {
            if (elect_one()) {     // both blocks' bytes are counted in the first one's barrier
              hdr->filled[stage] = round + 1u;
              if (rank == 0) mbar_arrive_expect_tx(full, 2 * S::kStageBytes);
              const uint32_t lead = map_to_cta(full, 0);
              tma_load_2d_pair(dst, &maps.a, lead, kb * 128, m_blk * 128);
              tma_load_2d_pair(dst + kABytes, &maps.b, lead, kb * 128, n_blk * BN + rank * (BN / 2));
              tma_load_2d_pair(sf, &maps.sfa, lead, kb * 256, m_blk);
              tma_load_2d_pair(sf + 1024, &maps.sfb, lead, kb * 256, n_blk * (BN / 128));
            }
          } else {
            const uint32_t sf_bytes = p.k_tiles - 2 * kb >= 2 ? 1024u : 512u;
            const int rt0 = n_blk * BN / 128;
            const int rts = S::kRowTiles < p.row_tiles_b - rt0 ? S::kRowTiles : p.row_tiles_b - rt0;
            if (elect_one()) {
              hdr->filled[stage] = round + 1u;
              mbar_arrive_expect_tx(full, kABytes + S::kBBytes + sf_bytes * (1 + rts));
              tma_load_2d(dst, &maps.a, full, kb * 128, m_blk * 128);
              tma_load_2d(dst + kABytes, &maps.b, full, kb * 128, n_blk * BN);
              bulk_load(sf, p.sfa + (static_cast<int64_t>(m_blk) * p.k_tiles + 2 * kb) * kTileBytes, sf_bytes, full);
              for (int i = 0; i < rts; ++i)
                bulk_load(sf + 1024 * (1 + i), p.sfb + (static_cast<int64_t>(rt0 + i) * p.k_tiles + 2 * kb) * kTileBytes, sf_bytes, full);
            }
          }
          __syncwarp();
        }
        if (++turn == turns) turn = 0;
        if (++stage == n_st) { stage = 0; ++round; }
      }
    }
    __syncwarp();
  } else if (warp == kProducers) {
    uint32_t stage = 0, phase = 0, buf = 0, bph = 0;
    bool ok = rank == 0;      // the first block of a pair issues for both
    for (int t = tile0; t < p.tiles && ok; t += tile_step) {
      const int n0 = (t % p.n_tiles) * BN;
      if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&hdr->d_empty[buf]), bph ^ 1u, abort_flag, 0x2200u | buf))) { ok = false; break; }
      tc_fence_after();
      const uint32_t d = tmem + buf * 128;
      for (int kb = 0; kb < k_stages; ++kb) {
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&hdr->full[stage]), phase, abort_flag, 0x2300u | stage))) { ok = false; break; }
        tc_fence_after();
        const uint32_t at = smem_u32(smem + stage * S::kStageBytes);
        const uint64_t a0 = make_smem_desc_sw128(at), b0 = make_smem_desc_sw128(at + kABytes);
        const uint64_t sf0 = scale_desc(at + kABytes + S::kBBytes);
        const uint32_t sfa = tmem + kSfCol + stage * S::kSfCols, sfb = sfa + 8;
        const int kts = p.k_tiles - 2 * kb < 2 ? p.k_tiles - 2 * kb : 2;
        if (elect_one()) {
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) {
            if (kt < kts) {   // a scale tile that is not there has no values either
              copy_scales<PAIR>(sfa + 4 * kt, sf0 + static_cast<uint64_t>(kt * (kTileBytes >> 4)));
#pragma unroll
              for (int i = 0; i < S::kRowTiles; ++i)
                copy_scales<PAIR>(sfb + (kt * S::kRowTiles + i) * 4, sf0 + static_cast<uint64_t>((1024 * (1 + i) + kt * kTileBytes) >> 4));
#pragma unroll
              for (int j = 0; j < 2; ++j)   // 64 k = 32 bytes inside the swizzled row
                mma_mxf4<PAIR>(d, a0 + static_cast<uint64_t>(4 * kt + 2 * j), b0 + static_cast<uint64_t>(4 * kt + 2 * j),
                               mxf4_idesc(PAIR ? 256 : 128, BN, j), sfa + 4 * kt,
                               sfb + kt * S::kRowTiles * 4 + (BN == 64 && (n0 & 64) ? 2 : 0), (kb || kt || j) ? 1u : 0u);
            }
          }
          commit<PAIR>(smem_u32(&hdr->empty[stage]));
        }
        __syncwarp();
        if (++stage == n_st) { stage = 0; phase ^= 1u; }
      }
      if (!ok) break;
      if (elect_one()) commit<PAIR>(smem_u32(&hdr->d_full[buf]));
      __syncwarp();
      if (++buf == S::kBufs) { buf = 0; bph ^= 1u; }
    }
  } else {
    const int ew = warp - kProducers - 1;
    const int quarter = warp & 3, sub = ew >> 2;   // pieces sub, sub + 2, ... of the tile's columns
    unsigned char* stage = staging + ew * kStagingBytes;
    float* my_bias = biases + ew * 128;
    constexpr int kMine = BN / 64;
    uint32_t buf = 0, bph = 0, piece = 0;
    bool ok = true;
    for (int t = tile0; t < p.tiles && ok; t += tile_step) {
      const int64_t n_first = static_cast<int64_t>(t % p.n_tiles) * BN;
      const int64_t row0 = (static_cast<int64_t>(PAIR ? 2 : 1) * (t / p.n_tiles) + rank) * 128 + quarter * 32;
      if (p.out.bias != nullptr) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          const int64_t n = n_first + (sub + 2 * i) * 32 + lane;
          my_bias[32 * i + lane] = n < p.out.cols ? load_as_float(p.out.bias, p.out.bias_dtype, n) : 0.0f;
        }
        __syncwarp();
      }
      const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
      float sum[kMine][32];
      const bool there = __all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&hdr->d_full[buf]), bph, abort_flag, 0x2500u | buf));
      if (there) {   // all of this warp's sums into registers: the accumulator is free before they are looked at
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < kMine; ++i) tmem_ld32(tmem + lanes + buf * 128 + (sub + 2 * i) * 32, reinterpret_cast<uint32_t(&)[32]>(sum[i]));
        tmem_ld_wait();
        tc_fence_before();
      }
      // The warps meet, whether they got there or not (all leave together), and one arrival stands for all: sixteen on one
      // barrier, half of them from the other block, held 18944 x 256 -> 2048 at 30 us (24).
      ok = all_agree(1, kEpiWarps * 32, there);
      if (!ok) break;
      if (ew == 0 && lane == 0) {
        if constexpr (PAIR) remote_arrive(map_to_cta(smem_u32(&hdr->d_empty[buf]), 0));
        else mbar_arrive(smem_u32(&hdr->d_empty[buf]));
      }
      __syncwarp();
      if (++buf == S::kBufs) { buf = 0; bph ^= 1u; }
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int64_t n0 = n_first + (sub + 2 * i) * 32;
        const float* bias = p.out.bias != nullptr ? my_bias + 32 * i : nullptr;
        if (row0 < p.out.rows && n0 < p.out.cols) put_chunk<ES>(sum[i], p.out, &maps.y, stage, piece, bias, row0, n0, lane);
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

// scale tiles as 32-bit words: [row tile][word], a stage's 256 words of one row tile (sfa) or two (sfb)
bool scale_map(CUtensorMap* m, const uint8_t* scales, int64_t rows, int64_t K, int box_tiles) {
  const cuuint64_t words = static_cast<cuuint64_t>(block_tiles(K)) * (kTileBytes / 4), pitch = words * 4;
  const cuuint64_t dims[2] = {words, static_cast<cuuint64_t>(row_tiles(rows))};
  const cuuint32_t box[2] = {256, static_cast<cuuint32_t>(box_tiles)};
  return encode_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, scales, dims, &pitch, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <int BN, int ES, bool PAIR>
int launch_gemm(const uint8_t* xc, const uint8_t* xs, const uint8_t* wc, const uint8_t* ws, const Out& out, int64_t K, cudaStream_t st) {
  using S = Shape<BN, PAIR>;
  GemmMaps maps;
  GemmParams p = {};
  p.sfa = xs;
  p.sfb = ws;
  p.out = out;
  p.k_tiles = static_cast<int>(block_tiles(K));
  p.row_tiles_b = static_cast<int>(row_tiles(out.cols));
  p.n_tiles = static_cast<int>((out.cols + BN - 1) / BN);
  const int64_t tiles = (PAIR ? (row_tiles(out.rows) + 1) / 2 : row_tiles(out.rows)) * p.n_tiles;
  if (tiles > 0x7FFFFFFF - kNumSMs) return DIMQ_ERR_TOO_LARGE;
  p.tiles = static_cast<int>(tiles);
  if (!code_map(&maps.a, xc, out.rows, K, 128) || !code_map(&maps.b, wc, out.cols, K, PAIR ? BN / 2 : BN) ||
      (out.tma && !encode_out(&maps.y, out)) ||
      (PAIR && (!scale_map(&maps.sfa, xs, out.rows, K, 1) || !scale_map(&maps.sfb, ws, out.cols, K, BN / 128))))
    return DIMQ_ERR_DRIVER;
  const size_t fixed = 1024 + kHeaderBytes + kBiasBytes + kEpiWarps * kStagingBytes;
  p.stages = static_cast<int>((kSmemMax - fixed) / S::kStageBytes);
  if (p.stages > S::kMost) p.stages = S::kMost;
  auto kern = mx_gemm_kernel<BN, ES, PAIR>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemMax));
  if (e != cudaSuccess) return static_cast<int>(e);
  const int64_t most = PAIR ? kNumSMs / 2 : kNumSMs;
  const unsigned grid = static_cast<unsigned>((tiles < most ? tiles : most) * (PAIR ? 2 : 1));
  e = launch_dependent(kern, grid, kThreads, fixed + p.stages * S::kStageBytes, st, PAIR ? 2 : 1, maps, p);
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
}

// Columns a tile takes (512: a pair of blocks): the form that needs the fewest waves of tiles, weighed by what a 256-k
// step of it costs.
int choose_bn(int64_t M, int64_t N) {
  const int form[4] = {512, 256, 128, 64};
  const double cost[4] = {600.0, 768.0, 520.0, 430.0};
  int best = 64;
  double least = 0.0;
  for (int i = 0; i < 4; ++i) {
    const int64_t width = form[i] > 256 ? 256 : form[i];
    const int64_t rows = form[i] > 256 ? (row_tiles(M) + 1) / 2 : row_tiles(M), side_by_side = form[i] > 256 ? kNumSMs / 2 : kNumSMs;
    const int64_t tiles = rows * ((N + width - 1) / width);
    const double c = static_cast<double>((tiles + side_by_side - 1) / side_by_side) * cost[i];
    if (i == 0 || c < least) { least = c; best = form[i]; }
  }
  return best;
}

int gemm(const uint8_t* xc, const uint8_t* xs, const uint8_t* wc, const uint8_t* ws, const Out& out, int64_t K, cudaStream_t st) {
  const int bn = choose_bn(out.rows, out.cols);
#define DIMQ_MX_GEMM(BN, PAIR)                                                                \
  return out.dtype == DIMQ_F32 ? launch_gemm<BN, 4, PAIR>(xc, xs, wc, ws, out, K, st)         \
                               : launch_gemm<BN, 2, PAIR>(xc, xs, wc, ws, out, K, st)
  if (bn == 512) DIMQ_MX_GEMM(256, true);
  if (bn == 256) DIMQ_MX_GEMM(256, false);
  if (bn == 128) DIMQ_MX_GEMM(128, false);
  DIMQ_MX_GEMM(64, false);
#undef DIMQ_MX_GEMM
}

int check_sizes(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N <= 0 || K <= 0) return DIMQ_ERR_BAD_SIZE;
  if (M > 0x7FFFFF00 || N > 0x7FFFFF00 || K > 0x7FFFFF00) return DIMQ_ERR_TOO_LARGE;
  return DIMQ_OK;
}

int64_t codes_room(int64_t M, int64_t K) { return (codes_bytes(M, K, DIMQ_MX_FP4) + 511) / 512 * 512; }

}  // namespace

int read_mx_status(uint32_t* status) { return tc::read_and_clear_device_status(status); }

}  // namespace dimq

using namespace dimq;

extern "C" int dimq_mx_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int coded, int64_t* bytes) {
  if (bytes == nullptr) return DIMQ_ERR_NULL_POINTER;
  *bytes = 0;
  const int rc = check_sizes(M, N, K);
  if (rc != DIMQ_OK) return rc;
  if (!coded && !mx_small_takes(M, N, K)) *bytes = codes_room(M, K) + mx::scales_bytes(M, K);
  return DIMQ_OK;
}

extern "C" int dimq_mx_linear(const void* x, int x_dtype, const uint8_t* x_scales, const uint8_t* w_codes, const uint8_t* w_scales,
                              const void* bias, int bias_dtype, const void* residual, void* y, int y_dtype, int64_t M, int64_t N,
                              int64_t K, int epilogue, void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_sizes(M, N, K);
  if (rc != DIMQ_OK) return rc;
  if ((x_scales == nullptr && !valid_dtype(x_dtype)) || !valid_dtype(y_dtype) || (bias != nullptr && !valid_dtype(bias_dtype))) return DIMQ_ERR_BAD_DTYPE;
  if (epilogue < DIMQ_EPI_NONE || epilogue > DIMQ_EPI_ADD_RELU) return DIMQ_ERR_UNSUPPORTED;
  if (M == 0) return DIMQ_OK;
  if (x == nullptr || w_codes == nullptr || w_scales == nullptr || y == nullptr) return DIMQ_ERR_NULL_POINTER;
  if (!aligned(w_codes, 16) || !aligned(w_scales, 16) || !aligned(workspace, 16) || !aligned(x_scales, 16) ||
      (x_scales != nullptr && !aligned(x, 16)))
    return DIMQ_ERR_ALIGNMENT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const uint8_t *xc = static_cast<const uint8_t*>(x), *xs = x_scales;
  if (x_scales == nullptr && mx_small_takes(M, N, K))
    return mx_small(x, x_dtype, w_codes, w_scales, bias, bias_dtype, residual, y, y_dtype, M, N, K, epilogue, st);
  if (x_scales == nullptr) {
    if (workspace == nullptr || workspace_bytes < codes_room(M, K) + mx::scales_bytes(M, K)) return DIMQ_ERR_SCRATCH_TOO_SMALL;
    uint8_t* c = static_cast<uint8_t*>(workspace);
    uint8_t* s = c + codes_room(M, K);
    rc = mx_quantize(x, x_dtype, M, K, c, s, nullptr, nullptr, st);
    if (rc != DIMQ_OK) return rc;
    xc = c;
    xs = s;
  }
  mx::Out out = {y, residual, bias, M, N, bias_dtype, y_dtype, epilogue, 0};
  out.tma = mx::out_by_map(out);
  return gemm(xc, xs, w_codes, w_scales, out, K, st);
}
