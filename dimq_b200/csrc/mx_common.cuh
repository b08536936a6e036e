// Microscaled (MX) numbers: 32 consecutive values of a row share a power of two.
//
// A block of 32 values v has the exponent E = max(floor(log2 max|v|) - emax, -127), stored as the byte E + 127, and one
// code per value, v * 2^-E rounded to nearest even and saturated:
//   fp4   e2m1 (0, .5, 1, 1.5, 2, 3, 4, 6 and sign), emax = 2; two codes to a byte, the first in the low half
//   int8  two's complement with 6 fraction bits, -127/64 .. 127/64, emax = 0
// The byte 255 says that the block held a NaN or an infinity: all of it reads as NaN.  A block of zeros has the byte 0.
// Scaling by a power of two is exact, so a code's value is what rounding to nearest in 64 bits gives.
//
// Codes are row-major, rows padded with zeros to whole blocks.  Scale bytes lie in tiles of 128 rows x 4 blocks,
// [row tile][block tile][row % 32][row / 32 % 4][block % 4]: 512 contiguous bytes that the tensor core's scale memory
// takes with one copy.  The padding of both dimensions is zero.
#pragma once

#include "common.cuh"

namespace dimq {
namespace mx {

constexpr int kBlock = 32;
constexpr int kTileBytes = 512;   // scales of 128 rows x 4 blocks

inline bool valid_format(int f) { return f == DIMQ_MX_FP4 || f == DIMQ_MX_INT8; }
__host__ __device__ inline int64_t blocks_of(int64_t cols) { return (cols + kBlock - 1) / kBlock; }
__host__ __device__ inline int64_t block_tiles(int64_t cols) { return (blocks_of(cols) + 3) / 4; }
__host__ __device__ inline int64_t row_tiles(int64_t rows) { return (rows + 127) / 128; }
inline int64_t codes_pitch(int64_t cols, int format) { return blocks_of(cols) * (format == DIMQ_MX_FP4 ? 16 : 32); }
inline int64_t codes_bytes(int64_t rows, int64_t cols, int format) { return rows * codes_pitch(cols, format); }
inline int64_t scales_bytes(int64_t rows, int64_t cols) { return row_tiles(rows) * block_tiles(cols) * kTileBytes; }

// byte of the block exponent from the largest |v| (as its bits); 255 where that is an infinity or a NaN
__device__ __forceinline__ uint32_t scale_byte(uint32_t top_bits, int emax) {
  const int field = static_cast<int>(top_bits >> 23);
  return field == 255 ? 255u : static_cast<uint32_t>(max(field - emax, 0));
}
// 2^(b - 127) and 2^(127 - b); exact, subnormal at one end each.  b = 255 reads as NaN.
__device__ __forceinline__ float scale_of(uint32_t b) {
  return __uint_as_float(b == 0u ? 0x00400000u : b == 255u ? 0x7FC00000u : b << 23);
}
__device__ __forceinline__ float inverse_scale(uint32_t b) {
  return __uint_as_float(b >= 254u ? 0x00400000u : (254u - b) << 23);
}

// two floats -> two e2m1 codes, `lo` in the low half; nearest even, saturating at 6
__device__ __forceinline__ uint32_t encode_fp4_pair(float lo, float hi) {
  uint32_t d;
  asm("{\n\t.reg .b8 b;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %1, %2;\n\tcvt.u32.u8 %0, b;\n\t}" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
template <typename T>
struct Eight {   // eight consecutive values as they are loaded
  uint4 q[sizeof(T) / 2];
};

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ row, int64_t k, int64_t cols, float (&v)[8]) {
  constexpr int kPer = 16 / sizeof(T);   // values per 16 bytes; rows are whole 16-byte pieces where VEC
  if (VEC) {
    Eight<T> e;
#pragma unroll
    for (int i = 0; i < 8 / kPer; ++i) {
      e.q[i] = make_uint4(0u, 0u, 0u, 0u);
      if (k + i * kPer < cols) e.q[i] = __ldg(reinterpret_cast<const uint4*>(row + k + i * kPer));
    }
    const T* p = reinterpret_cast<const T*>(&e);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float<T>(p[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < cols ? to_float<T>(row[k + i]) : 0.0f;
  }
}

// bits of the largest |v| of a block that four neighbouring lanes hold, eight values each
__device__ __forceinline__ uint32_t block_top(const float (&v)[8]) {
  uint32_t top = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
  return max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
}
// eight values of a block whose scale byte is b -> codes
__device__ __forceinline__ uint32_t encode_fp4(const float (&v)[8], uint32_t b) {
  const float f = inverse_scale(b);
  uint32_t w = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= encode_fp4_pair(v[2 * i] * f, v[2 * i + 1] * f) << (8 * i);
  return b == 255u ? 0u : w;
}
// eight e2m1 codes -> floats.  A code's three bits, moved to a half's lowest exponent bits and highest mantissa bit, are
// its magnitude times 2^-14, subnormal code and all.
__device__ __forceinline__ void decode_fp4(uint32_t w, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint32_t c = (w >> (4 * i)) & 0xFFu;
    const uint32_t h = ((c & 0x7u) << 9) | ((c & 0x8u) << 12) | ((c & 0x70u) << 21) | ((c & 0x80u) << 24);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    v[i] = f.x * 16384.0f;
    v[i + 1] = f.y * 16384.0f;
  }
}
__device__ __forceinline__ void decode_int8(uint2 w, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t word = i < 4 ? w.x : w.y;
    v[i] = static_cast<float>(static_cast<int8_t>(word >> (8 * (i & 3)))) * 0.015625f;
  }
}

__host__ __device__ __forceinline__ int64_t scale_offset(int64_t row, int64_t block, int64_t tiles) {
  return ((row >> 7) * tiles + (block >> 2)) * kTileBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

}  // namespace mx
}  // namespace dimq
