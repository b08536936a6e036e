// The gradients of the microscaled linear layer.
//
// One plain kernel for both: 64 x 64 tiles of the result, 16 of the reduction at a time decoded to fp32 in shared
// memory, 4 x 4 results a thread.
#include "mx_common.cuh"

namespace dimq {
namespace {

using namespace mx;

struct Coded {   // a microscaled matrix [rows][cols]
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t blocks, tiles;
  int fp4;
  __device__ float at(int64_t r, int64_t k) const {
    const float f = scale_of(scales[scale_offset(r, k >> 5, tiles)]);
    float v[8];
    if (fp4) {
      decode_fp4(codes[r * blocks * 16 + (k >> 1)] >> (4 * (k & 1)), v);
      return v[0] * f;
    }
    return static_cast<float>(static_cast<int8_t>(codes[r * blocks * 32 + k])) * 0.015625f * f;
  }
};
Coded coded(const void* codes, const uint8_t* scales, int64_t cols, int format) {
  return {static_cast<const uint8_t*>(codes), scales, blocks_of(cols), block_tiles(cols), format == DIMQ_MX_FP4};
}

struct Dense {
  const void* p;
  int dtype;
  int64_t cols;
  __device__ float at(int64_t r, int64_t k) const { return load_as_float(p, dtype, r * cols + k); }
};

// c[r][j] = sum_t A(r, t) B(t, j); AT / BT: the operand is stored with its axes exchanged
template <typename A, bool AT, typename B, bool BT>
__global__ void __launch_bounds__(256)
mx_plain_kernel(A a, B b, int64_t R, int64_t J, int64_t T, const void* bias, int bias_dtype, const void* residual, void* c,
                int c_dtype, int epilogue) {
  __shared__ float sa[16][65], sb[16][65];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * 64, j0 = static_cast<int64_t>(blockIdx.x) * 64;
  float acc[4][4] = {};
  for (int64_t t0 = 0; t0 < T; t0 += 16) {
    for (int i = threadIdx.x; i < 1024; i += 256) {
      const int t = AT ? i >> 6 : i & 15, r = AT ? i & 63 : i >> 4;
      const bool in = r0 + r < R && t0 + t < T;
      sa[t][r] = in ? (AT ? a.at(t0 + t, r0 + r) : a.at(r0 + r, t0 + t)) : 0.0f;
      const int tb = BT ? i & 15 : i >> 6, j = BT ? i >> 4 : i & 63;
      const bool inb = j0 + j < J && t0 + tb < T;
      sb[tb][j] = inb ? (BT ? b.at(j0 + j, t0 + tb) : b.at(t0 + tb, j0 + j)) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 16; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[t][ty + 16 * i], sb[t][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t r = r0 + ty + 16 * i, k = j0 + tx + 16 * j;
      if (r >= R || k >= J) continue;
      float v = acc[i][j];
      if (bias != nullptr) v += load_as_float(bias, bias_dtype, k);
      v = finish_value(v, epilogue, residual != nullptr, residual != nullptr ? load_as_float(residual, c_dtype, r * J + k) : 0.0f);
      store_from_float(c, c_dtype, r * J + k, v);
    }
}

__global__ void __launch_bounds__(256)
mx_column_sum_kernel(Dense a, int64_t rows, void* out, int out_dtype) {
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x & 31);
  __shared__ float part[8][32];
  float s = 0.0f;
  if (j < a.cols)
    for (int64_t r = threadIdx.x >> 5; r < rows; r += 8) s += a.at(r, j);
  part[threadIdx.x >> 5][threadIdx.x & 31] = s;
  __syncthreads();
  if (threadIdx.x < 32 && j < a.cols) {
    for (int i = 1; i < 8; ++i) s += part[i][threadIdx.x];
    store_from_float(out, out_dtype, j, s);
  }
}

template <typename A, bool AT, typename B, bool BT>
int plain(A a, B b, int64_t R, int64_t J, int64_t T, const void* bias, int bias_dtype, const void* residual, void* c, int c_dtype,
          int epilogue, cudaStream_t st) {
  const int64_t gx = (J + 63) / 64, gy = (R + 63) / 64;
  if (gx > 0x7FFFFFFF || gy > 65535) return DIMQ_ERR_TOO_LARGE;
  mx_plain_kernel<A, AT, B, BT><<<dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy)), 256, 0, st>>>(
      a, b, R, J, T, bias, bias_dtype, residual, c, c_dtype, epilogue);
  return launch_status();
}

int check_sizes(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N <= 0 || K <= 0) return DIMQ_ERR_BAD_SIZE;
  if (M > 0x7FFFFF00 || N > 0x7FFFFF00 || K > 0x7FFFFF00) return DIMQ_ERR_TOO_LARGE;
  return DIMQ_OK;
}

}  // namespace
}  // namespace dimq

using namespace dimq;

extern "C" int dimq_mx_grad_input(const void* dy, int dy_dtype, const uint8_t* w_codes, const uint8_t* w_scales, void* dx,
                                  int dx_dtype, int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  const int rc = check_sizes(M, N, K);
  if (rc != DIMQ_OK) return rc;
  if (!valid_dtype(dy_dtype) || !valid_dtype(dx_dtype)) return DIMQ_ERR_BAD_DTYPE;
  if (M == 0) return DIMQ_OK;
  if (dy == nullptr || w_codes == nullptr || w_scales == nullptr || dx == nullptr) return DIMQ_ERR_NULL_POINTER;
  if (!aligned(w_codes, 16) || !aligned(w_scales, 16) || !aligned(workspace, 16)) return DIMQ_ERR_ALIGNMENT;
  int64_t need = 0;
  dimq_mx_grad_workspace_bytes(dy_dtype, M, N, K, &need);
  if (workspace == nullptr || workspace_bytes < need) return DIMQ_ERR_SCRATCH_TOO_SMALL;
  return plain<Dense, false, Coded, false>(Dense{dy, dy_dtype, N}, coded(w_codes, w_scales, K, DIMQ_MX_FP4), M, K, N, nullptr, 0,
                                           nullptr, dx, dx_dtype, DIMQ_EPI_NONE, static_cast<cudaStream_t>(stream));
}

extern "C" int dimq_mx_grad_weight(const void* dy, int dy_dtype, const void* x_codes, const uint8_t* x_scales, int format, void* dw,
                                   int dw_dtype, void* db, int db_dtype, int64_t M, int64_t N, int64_t K, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  int rc = check_sizes(M, N, K);
  if (rc != DIMQ_OK) return rc;
  if (!mx::valid_format(format)) return DIMQ_ERR_BAD_BITS;
  if (!valid_dtype(dy_dtype) || (dw != nullptr && !valid_dtype(dw_dtype)) || (db != nullptr && !valid_dtype(db_dtype))) return DIMQ_ERR_BAD_DTYPE;
  if ((dw == nullptr && db == nullptr) || (M > 0 && (dy == nullptr || (dw != nullptr && (x_codes == nullptr || x_scales == nullptr))))) return DIMQ_ERR_NULL_POINTER;
  if (!aligned(x_codes, 16) || !aligned(x_scales, 16) || !aligned(workspace, 16)) return DIMQ_ERR_ALIGNMENT;
  int64_t need = 0;
  dimq_mx_grad_workspace_bytes(dy_dtype, M, N, K, &need);
  if (workspace == nullptr || workspace_bytes < need) return DIMQ_ERR_SCRATCH_TOO_SMALL;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dw != nullptr)
    rc = plain<Dense, true, Coded, false>(Dense{dy, dy_dtype, N}, coded(x_codes, x_scales, K, format), N, K, M, nullptr, 0, nullptr, dw,
                                        dw_dtype, DIMQ_EPI_NONE, st);
  if (rc != DIMQ_OK || db == nullptr) return rc;
  mx_column_sum_kernel<<<static_cast<unsigned>((N + 31) / 32), 256, 0, st>>>(Dense{dy, dy_dtype, N}, M, db, db_dtype);
  return launch_status();
}

extern "C" int dimq_mx_grad_workspace_bytes(int dy_dtype, int64_t M, int64_t N, int64_t K, int64_t* bytes) {
  if (bytes == nullptr) return DIMQ_ERR_NULL_POINTER;
  *bytes = 0;
  if (!valid_dtype(dy_dtype)) return DIMQ_ERR_BAD_DTYPE;
  const int rc = check_sizes(M, N, K);
  if (rc == DIMQ_OK) *bytes = 16;
  return rc;
}
