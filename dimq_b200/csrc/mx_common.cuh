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

// packed pairs of fp32
__device__ __forceinline__ float2 mul2(float2 a, float b) {
  uint64_t d, x, y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %1};" : "=l"(y) : "f"(b));
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(x), "l"(y));
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(d));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float b) {
  uint64_t d, x, y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %1};" : "=l"(y) : "f"(b));
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(x), "l"(y));
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(d));
  return r;
}

// Eight consecutive values of a row as they are stored: what a lane holds of a block, four lanes to a block.
template <typename T>
struct Eight {
  uint32_t w[2 * sizeof(T)];
};
template <typename T>
__device__ __forceinline__ Eight<T> no_values() {
  Eight<T> e;
#pragma unroll
  for (int i = 0; i < static_cast<int>(2 * sizeof(T)); ++i) e.w[i] = 0u;
  return e;
}
// rows of whole 16-byte pieces
template <typename T>
__device__ __forceinline__ Eight<T> load_pieces(const T* __restrict__ row, int64_t k, int64_t cols) {
  constexpr int kPer = 16 / sizeof(T);
  Eight<T> e = no_values<T>();
#pragma unroll
  for (int i = 0; i < 8 / kPer; ++i)
    if (k + i * kPer < cols) *reinterpret_cast<uint4*>(&e.w[4 * i]) = __ldg(reinterpret_cast<const uint4*>(row + k + i * kPer));
  return e;
}
// any row: the warp reads neighbours (32 values at a time) and the values change hands in shared memory, `swap` 256 of
// them; k0 is the first of the warp's 256.
template <typename T>
__device__ __forceinline__ void load_neighbours(const T* __restrict__ row, int64_t k0, int64_t cols, int lane, T (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t k = k0 + 32 * i + lane;
    v[i] = k < cols ? row[k] : from_float<T>(0.0f);
  }
}
template <typename T>
__device__ __forceinline__ Eight<T> change_hands(const T (&v)[8], T* swap, int lane) {
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) swap[32 * i + lane] = v[i];
  __syncwarp();
  Eight<T> e;
  const uint4* from = reinterpret_cast<const uint4*>(swap + 8 * lane);
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) *reinterpret_cast<uint4*>(&e.w[4 * i]) = from[i];
  return e;
}

__device__ __forceinline__ float2 pair_of(const Eight<float>& e, int i) {
  return make_float2(__uint_as_float(e.w[2 * i]), __uint_as_float(e.w[2 * i + 1]));
}
__device__ __forceinline__ float2 pair_of(const Eight<__half>& e, int i) { return __half22float2(*reinterpret_cast<const __half2*>(&e.w[i])); }
__device__ __forceinline__ float2 pair_of(const Eight<__nv_bfloat16>& e, int i) {
  return make_float2(__uint_as_float(e.w[i] << 16), __uint_as_float(e.w[i] & 0xFFFF0000u));
}

// bits (as fp32) of the largest |v| of a block; among bits without the sign a NaN is larger than an infinity, and that
// larger than any number, in every type
__device__ __forceinline__ uint32_t block_top(const Eight<float>& e) {
  uint32_t top = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, e.w[i] & 0x7FFFFFFFu);
  top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
  return max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
}
__device__ __forceinline__ uint32_t top_of_pairs(const uint32_t (&w)[4]) {
  uint32_t top = w[0] & 0x7FFF7FFFu;
#pragma unroll
  for (int i = 1; i < 4; ++i) top = __vmaxu2(top, w[i] & 0x7FFF7FFFu);
  top = __vmaxu2(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
  top = __vmaxu2(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
  return max(top & 0xFFFFu, top >> 16);
}
__device__ __forceinline__ uint32_t block_top(const Eight<__nv_bfloat16>& e) { return top_of_pairs(e.w) << 16; }
__device__ __forceinline__ uint32_t block_top(const Eight<__half>& e) {
  return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(top_of_pairs(e.w)))));
}

// eight values of a block whose scale byte is b -> e2m1 codes, nearest even, saturating at 6
template <typename T>
__device__ __forceinline__ uint32_t encode_fp4(const Eight<T>& e, uint32_t b) {
  const float f = inverse_scale(b);
  float2 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = mul2(pair_of(e, i), f);
  uint32_t d;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(d) : "f"(v[0].x), "f"(v[0].y), "f"(v[1].x), "f"(v[1].y), "f"(v[2].x), "f"(v[2].y), "f"(v[3].x), "f"(v[3].y));
  return b == 255u ? 0u : d;
}
// ... -> multiples of 1/64.  Adding 1.5 * 2^23 rounds to the nearest even integer and leaves it in the low byte.
template <typename T>
__device__ __forceinline__ uint2 encode_int8(const Eight<T>& e, uint32_t b) {
  const float f = inverse_scale(b);
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 v = mul2(mul2(pair_of(e, i), f), 64.0f);
    v = add2(make_float2(fminf(fmaxf(v.x, -127.0f), 127.0f), fminf(fmaxf(v.y, -127.0f), 127.0f)), 12582912.0f);
    c[2 * i] = __float_as_uint(v.x);
    c[2 * i + 1] = __float_as_uint(v.y);
  }
  uint2 d;
  d.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
  d.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
  return b == 255u ? make_uint2(0u, 0u) : d;
}

// eight e2m1 codes -> their values times f
__device__ __forceinline__ void decode_fp4(uint32_t w, float f, float2 (&v)[4]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = mul2(__half22float2(*reinterpret_cast<const __half2*>(&h[i])), f);
}
// eight 8-bit codes -> their values times f.  A byte with its sign bit turned, under the exponent of 2^23, is 2^23 + 128 + code.
__device__ __forceinline__ void decode_int8(uint2 w, float f, float2 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t word = (i < 2 ? w.x : w.y) ^ 0x80808080u;
    const float2 c = make_float2(__uint_as_float(__byte_perm(word, 0x4B000000u, i & 1 ? 0x7542 : 0x7540)),
                                 __uint_as_float(__byte_perm(word, 0x4B000000u, i & 1 ? 0x7543 : 0x7541)));
    v[i] = mul2(mul2(add2(c, -8388736.0f), 0.015625f), f);
  }
}

// programmatic dependents of this grid may start; what it writes is theirs after their own wait
__device__ __forceinline__ void let_dependents_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace mx
}  // namespace dimq
