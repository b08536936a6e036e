// Quantisation to microscaled blocks and back (mx_common.cuh has the formats).  Both are one pass over memory: four
// lanes hold a block, eight values each, its largest magnitude takes two shuffles, and the rest is conversions.
//
// A warp takes the same 256 features of the rows r, r + 32, r + 64 and r + 96 of a row tile: four loads of 16 bytes a
// lane in flight (fp32: eight), and the scale bytes of the four rows are the 16 that lie together in the tile.  Rows that
// do not start on 16 bytes are read and written 32 neighbours at a time and change hands in shared memory.
#include "mx_common.cuh"

namespace dimq {
namespace {

using namespace mx;

constexpr int kThreads = 256;
constexpr int kSpan = 256;        // features a warp takes at a time
constexpr int kRowsPerBlock = 8;  // rows r of one row tile, each with its three rows 32 further

// the four bytes of a half warp's blocks in one word, known to all its lanes
__device__ __forceinline__ uint32_t gather_bytes(uint32_t b, int lane) {
  uint32_t w = b << (8 * ((lane >> 2) & 3));
  w |= __shfl_xor_sync(0xFFFFFFFFu, w, 4);
  w |= __shfl_xor_sync(0xFFFFFFFFu, w, 8);
  return w;
}

// C4 / C8: the formats written
template <typename T, bool VEC, bool C4, bool C8>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 && VEC ? 6 : 1)   // 42 registers: 11008 x 4096 bf16 25 -> 22 us (fp32: slower)
mx_quantize_kernel(const T* __restrict__ x, int64_t rows, int64_t cols, int64_t spans, uint8_t* __restrict__ codes4,
                   uint8_t* __restrict__ scales4, uint8_t* __restrict__ codes8, uint8_t* __restrict__ scales8) {
  __shared__ __align__(16) unsigned char swap[VEC ? 16 : 8 * kSpan * sizeof(T)];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t group = static_cast<int64_t>(blockIdx.x) / spans, span = static_cast<int64_t>(blockIdx.x) - group * spans;
  const int64_t tile = group >> 2;
  const int r = static_cast<int>(group & 3) * kRowsPerBlock + warp;
  const int64_t row0 = tile * 128 + r;
  const int64_t k = span * kSpan + lane * 8;
  const int64_t blocks = blocks_of(cols), tiles = block_tiles(cols);
  Eight<T> e[4];
  let_dependents_start();
  if constexpr (VEC) {
#pragma unroll
    for (int q = 0; q < 4; ++q) e[q] = row0 + 32 * q < rows ? load_pieces<T>(x + (row0 + 32 * q) * cols, k, cols) : no_values<T>();
  } else {
    T v[4][8];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      load_neighbours<T>(x + (row0 + 32 * q) * cols, span * kSpan, row0 + 32 * q < rows ? cols : 0, lane, v[q]);
#pragma unroll
    for (int q = 0; q < 4; ++q) e[q] = change_hands<T>(v[q], reinterpret_cast<T*>(swap) + warp * kSpan, lane);
  }
  uint32_t s4[4], s8[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t top = block_top(e[q]);
    const int64_t row = row0 + 32 * q;
    const bool write = row < rows && k < blocks * kBlock;
    if (C4) {
      const uint32_t b = scale_byte(top, 2), w = encode_fp4(e[q], b);
      if (write) *reinterpret_cast<uint32_t*>(codes4 + row * blocks * 16 + (k >> 1)) = w;
      s4[q] = gather_bytes(b, lane);
    }
    if (C8) {
      const uint32_t b = scale_byte(top, 0);
      const uint2 w = encode_int8(e[q], b);
      if (write) *reinterpret_cast<uint2*>(codes8 + row * blocks * 32 + k) = w;
      s8[q] = gather_bytes(b, lane);
    }
  }
  const int64_t block_tile = span * 2 + (lane >> 4);
  if ((lane & 15) == 0 && block_tile < tiles) {
    const int64_t at = (tile * tiles + block_tile) * kTileBytes + r * 16;
    if (C4) *reinterpret_cast<uint4*>(scales4 + at) = make_uint4(s4[0], s4[1], s4[2], s4[3]);
    if (C8) *reinterpret_cast<uint4*>(scales8 + at) = make_uint4(s8[0], s8[1], s8[2], s8[3]);
  }
}

template <typename T>
__device__ __forceinline__ Eight<T> pack_values(const float2 (&v)[4]);
template <>
__device__ __forceinline__ Eight<float> pack_values<float>(const float2 (&v)[4]) {
  Eight<float> e;
#pragma unroll
  for (int i = 0; i < 4; ++i) { e.w[2 * i] = __float_as_uint(v[i].x); e.w[2 * i + 1] = __float_as_uint(v[i].y); }
  return e;
}
template <>
__device__ __forceinline__ Eight<__half> pack_values<__half>(const float2 (&v)[4]) {
  Eight<__half> e;
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(e.w[i]) : "f"(v[i].y), "f"(v[i].x));
  return e;
}
template <>
__device__ __forceinline__ Eight<__nv_bfloat16> pack_values<__nv_bfloat16>(const float2 (&v)[4]) {
  Eight<__nv_bfloat16> e;
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(e.w[i]) : "f"(v[i].y), "f"(v[i].x));
  return e;
}

// Without PANELS out is [rows][cols].  With them it is [columns / 64][rows][64], zeros behind the last column: what TMA
// takes as boxes of 64 columns.  fill: columns written (cols, or the panels' 64s).
template <typename T, bool VEC, bool FP4, bool PANELS>
__global__ void __launch_bounds__(kThreads, VEC && !FP4 ? 6 : 1)              // 8192 x 4096 int8 19 -> 17 us (fp4: no gain)
mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows, int64_t cols,
                     int64_t spans, T* __restrict__ out, int64_t fill) {
  __shared__ __align__(16) unsigned char swap[VEC ? 16 : 8 * kSpan * sizeof(T)];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t group = static_cast<int64_t>(blockIdx.x) / spans, span = static_cast<int64_t>(blockIdx.x) - group * spans;
  const int64_t tile = group >> 2;
  const int r = static_cast<int>(group & 3) * kRowsPerBlock + warp;
  const int64_t row0 = tile * 128 + r;
  const int64_t k = span * kSpan + lane * 8;
  const int64_t blocks = blocks_of(cols), tiles = block_tiles(cols);
  const bool have = k < blocks * kBlock;
  uint2 w[4];
  uint4 s = make_uint4(0u, 0u, 0u, 0u);
  if (PANELS) let_dependents_start();
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    w[q] = make_uint2(0u, 0u);
    const int64_t row = row0 + 32 * q;
    if (have && row < rows) {
      if (FP4) w[q].x = __ldg(reinterpret_cast<const uint32_t*>(codes + row * blocks * 16 + (k >> 1)));
      else w[q] = __ldg(reinterpret_cast<const uint2*>(codes + row * blocks * 32 + k));
    }
  }
  if (have) s = __ldg(reinterpret_cast<const uint4*>(scales + (tile * tiles + span * 2 + (lane >> 4)) * kTileBytes + r * 16));
  const int sh = 8 * ((lane >> 2) & 3);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int64_t row = row0 + 32 * q;
    if (row >= rows) continue;        // the warp's
    const float f = scale_of(((q == 0 ? s.x : q == 1 ? s.y : q == 2 ? s.z : s.w) >> sh) & 0xFFu);
    float2 v[4];
    if (FP4) decode_fp4(w[q].x, f, v);
    else decode_int8(w[q], f, v);
    if (PANELS && k + 8 > cols) {     // a block that reads as NaN ends where the row does
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (k + 2 * i >= cols) v[i].x = 0.0f;
        if (k + 2 * i + 1 >= cols) v[i].y = 0.0f;
      }
    }
    const Eight<T> e = pack_values<T>(v);
    if constexpr (VEC && sizeof(T) == 4) {
      // two lanes exchange halves, so that each store of the warp writes whole sectors: the 32 bytes of the even lanes'
      // values, then those of the odd lanes'
      const bool odd = lane & 1;
      uint32_t mine[4], theirs[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        theirs[i] = __shfl_xor_sync(0xFFFFFFFFu, odd ? e.w[i] : e.w[4 + i], 1);
        mine[i] = odd ? e.w[4 + i] : e.w[i];
      }
      const int64_t base = k - (odd ? 8 : 0) + (odd ? 4 : 0);   // even lane: its first half; odd lane: the even lane's second
      T* dst = out + row * cols;
      if (base < fill) *reinterpret_cast<uint4*>(dst + base) = odd ? make_uint4(theirs[0], theirs[1], theirs[2], theirs[3]) : make_uint4(mine[0], mine[1], mine[2], mine[3]);
      if (base + 8 < fill) *reinterpret_cast<uint4*>(dst + base + 8) = odd ? make_uint4(mine[0], mine[1], mine[2], mine[3]) : make_uint4(theirs[0], theirs[1], theirs[2], theirs[3]);
    } else if constexpr (VEC) {
      T* dst = PANELS ? out + ((k >> 6) * rows + row) * 64 + (k & 63) : out + row * cols + k;
      constexpr int kPer = 16 / sizeof(T);
#pragma unroll
      for (int i = 0; i < 8 / kPer; ++i)
        if (k + i * kPer < fill) *reinterpret_cast<uint4*>(dst + i * kPer) = make_uint4(e.w[4 * i], e.w[4 * i + 1], e.w[4 * i + 2], e.w[4 * i + 3]);
    } else {                          // the values change hands, so that the warp stores neighbours
      T* mine = reinterpret_cast<T*>(swap) + warp * kSpan;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
        reinterpret_cast<uint4*>(mine + 8 * lane)[i] = make_uint4(e.w[4 * i], e.w[4 * i + 1], e.w[4 * i + 2], e.w[4 * i + 3]);
      __syncwarp();
      T* dst = out + row * cols;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t c = span * kSpan + 32 * i + lane;
        if (c < cols) dst[c] = mine[32 * i + lane];
      }
    }
  }
}

int grid_of(int64_t rows, int64_t width, int64_t* spans, unsigned* grid) {
  *spans = (width + kSpan - 1) / kSpan;
  const int64_t g = row_tiles(rows) * 4 * *spans;
  if (g > 0x7FFFFFFF) return DIMQ_ERR_TOO_LARGE;
  *grid = static_cast<unsigned>(g);
  return DIMQ_OK;
}

template <typename T>
int quantize_as(const void* x, int64_t rows, int64_t cols, void* c4, uint8_t* s4, void* c8, uint8_t* s8, cudaStream_t st) {
  int64_t spans;
  unsigned grid;
  // whole tiles of 4 blocks, so that the padding's scale bytes are written too
  const int rc = grid_of(rows, block_tiles(cols) * 128, &spans, &grid);
  if (rc != DIMQ_OK) return rc;
  const T* in = static_cast<const T*>(x);
  uint8_t *o4 = static_cast<uint8_t*>(c4), *o8 = static_cast<uint8_t*>(c8);
  const bool vec = aligned(x, 16) && (cols * static_cast<int64_t>(sizeof(T))) % 16 == 0;
#define DIMQ_MX_Q(V, A, B) mx_quantize_kernel<T, V, A, B><<<grid, kThreads, 0, st>>>(in, rows, cols, spans, o4, s4, o8, s8)
  if (c4 != nullptr && c8 != nullptr) { if (vec) DIMQ_MX_Q(true, true, true); else DIMQ_MX_Q(false, true, true); }
  else if (c4 != nullptr) { if (vec) DIMQ_MX_Q(true, true, false); else DIMQ_MX_Q(false, true, false); }
  else { if (vec) DIMQ_MX_Q(true, false, true); else DIMQ_MX_Q(false, false, true); }
#undef DIMQ_MX_Q
  return launch_status();
}

template <typename T, bool PANELS>
int dequantize_as(const void* codes, const uint8_t* scales, int format, int64_t rows, int64_t cols, void* out, cudaStream_t st) {
  int64_t spans;
  unsigned grid;
  const int64_t fill = PANELS ? (cols + 63) / 64 * 64 : cols;
  const int rc = grid_of(rows, fill, &spans, &grid);
  if (rc != DIMQ_OK) return rc;
  const uint8_t* in = static_cast<const uint8_t*>(codes);
  T* o = static_cast<T*>(out);
  const bool vec = PANELS || (aligned(out, 16) && (cols * static_cast<int64_t>(sizeof(T))) % 16 == 0);
#define DIMQ_MX_D(V, F) mx_dequantize_kernel<T, V, F, PANELS><<<grid, kThreads, 0, st>>>(in, scales, rows, cols, spans, o, fill)
  if (format == DIMQ_MX_FP4) { if (vec) DIMQ_MX_D(true, true); else DIMQ_MX_D(PANELS, true); }
  else { if (vec) DIMQ_MX_D(true, false); else DIMQ_MX_D(PANELS, false); }
#undef DIMQ_MX_D
  return launch_status();
}

}  // namespace

// x -> 4-bit codes, 8-bit codes, or both from one read (null: not wanted)
int mx_quantize(const void* x, int x_dtype, int64_t rows, int64_t cols, void* c4, uint8_t* s4, void* c8, uint8_t* s8,
                cudaStream_t st) {
  if (x_dtype == DIMQ_F32) return quantize_as<float>(x, rows, cols, c4, s4, c8, s8, st);
  if (x_dtype == DIMQ_F16) return quantize_as<__half>(x, rows, cols, c4, s4, c8, s8, st);
  return quantize_as<__nv_bfloat16>(x, rows, cols, c4, s4, c8, s8, st);
}

int mx_dequantize(const void* codes, const uint8_t* scales, int format, int64_t rows, int64_t cols, void* out, int out_dtype,
                  cudaStream_t st) {
  if (out_dtype == DIMQ_F32) return dequantize_as<float, false>(codes, scales, format, rows, cols, out, st);
  if (out_dtype == DIMQ_F16) return dequantize_as<__half, false>(codes, scales, format, rows, cols, out, st);
  return dequantize_as<__nv_bfloat16, false>(codes, scales, format, rows, cols, out, st);
}

// the same as bf16 panels [ceil(cols / 64)][rows][64], 16-byte aligned
int mx_decode_panels(const void* codes, const uint8_t* scales, int format, int64_t rows, int64_t cols, void* out, cudaStream_t st) {
  return dequantize_as<__nv_bfloat16, true>(codes, scales, format, rows, cols, out, st);
}

}  // namespace dimq

using namespace dimq;

static int check_mx(int64_t rows, int64_t cols, int format) {
  if (!mx::valid_format(format)) return DIMQ_ERR_BAD_BITS;
  if (rows < 0 || cols <= 0) return DIMQ_ERR_BAD_SIZE;
  if (cols > (int64_t(1) << 40) || rows > (int64_t(1) << 40) || (rows > 0 && cols > (int64_t(1) << 46) / rows)) return DIMQ_ERR_TOO_LARGE;
  return DIMQ_OK;
}

extern "C" int dimq_mx_sizes(int64_t rows, int64_t cols, int format, int64_t* code_bytes_per_row, int64_t* scale_bytes) {
  if (code_bytes_per_row == nullptr || scale_bytes == nullptr) return DIMQ_ERR_NULL_POINTER;
  const int rc = check_mx(rows, cols, format);
  if (rc != DIMQ_OK) return rc;
  *code_bytes_per_row = mx::codes_pitch(cols, format);
  *scale_bytes = mx::scales_bytes(rows, cols);
  return DIMQ_OK;
}

extern "C" int dimq_mx_quantize(const void* x, int x_dtype, int64_t rows, int64_t cols, int format, void* codes,
                                uint8_t* scales, void* stream) {
  if (!valid_dtype(x_dtype)) return DIMQ_ERR_BAD_DTYPE;
  const int rc = check_mx(rows, cols, format);
  if (rc != DIMQ_OK) return rc;
  if (rows == 0) return DIMQ_OK;
  if (x == nullptr || codes == nullptr || scales == nullptr) return DIMQ_ERR_NULL_POINTER;
  if (!aligned(codes, 16) || !aligned(scales, 16)) return DIMQ_ERR_ALIGNMENT;
  const bool four = format == DIMQ_MX_FP4;
  return mx_quantize(x, x_dtype, rows, cols, four ? codes : nullptr, four ? scales : nullptr, four ? nullptr : codes,
                     four ? nullptr : scales, static_cast<cudaStream_t>(stream));
}

extern "C" int dimq_mx_quantize_both(const void* x, int x_dtype, int64_t rows, int64_t cols, uint8_t* codes4, uint8_t* scales4,
                                     int8_t* codes8, uint8_t* scales8, void* stream) {
  if (!valid_dtype(x_dtype)) return DIMQ_ERR_BAD_DTYPE;
  const int rc = check_mx(rows, cols, DIMQ_MX_INT8);
  if (rc != DIMQ_OK) return rc;
  if (rows == 0) return DIMQ_OK;
  if (x == nullptr || codes4 == nullptr || scales4 == nullptr || codes8 == nullptr || scales8 == nullptr) return DIMQ_ERR_NULL_POINTER;
  if (!aligned(codes4, 16) || !aligned(scales4, 16) || !aligned(codes8, 16) || !aligned(scales8, 16)) return DIMQ_ERR_ALIGNMENT;
  return mx_quantize(x, x_dtype, rows, cols, codes4, scales4, codes8, scales8, static_cast<cudaStream_t>(stream));
}

extern "C" int dimq_mx_dequantize(const void* codes, const uint8_t* scales, int format, int64_t rows, int64_t cols, void* out,
                                  int out_dtype, void* stream) {
  if (!valid_dtype(out_dtype)) return DIMQ_ERR_BAD_DTYPE;
  const int rc = check_mx(rows, cols, format);
  if (rc != DIMQ_OK) return rc;
  if (rows == 0) return DIMQ_OK;
  if (codes == nullptr || scales == nullptr || out == nullptr) return DIMQ_ERR_NULL_POINTER;
  if (!aligned(codes, 16) || !aligned(scales, 16)) return DIMQ_ERR_ALIGNMENT;
  return mx_dequantize(codes, scales, format, rows, cols, out, out_dtype, static_cast<cudaStream_t>(stream));
}
