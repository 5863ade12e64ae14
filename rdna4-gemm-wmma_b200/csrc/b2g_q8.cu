// Matrix products of the 8-bit linear layer: the scaled 8-bit product and the weight gradient from
// an 8-bit checkpoint.
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/b2g_gemm.h"
#include "errors.h"
#include "host.h"
#include "q8.cuh"

namespace b2g {

namespace {

using namespace q8;

constexpr int kTile = 16;

// Any alignment and size: 16 x 16 tiles of C through shared memory, one element per thread.
// int8 sums are int32; e4m3 sums fp32, K in ascending order.
template <bool I8>
__global__ void __launch_bounds__(kTile* kTile)
    gemm_q8_generic_kernel(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K,
                           int64_t lda, int64_t ldb, int64_t ldc, const float* a_scale,
                           const float* b_scale, const float* bias, int c_dtype) {
  using T = typename std::conditional<I8, int, float>::type;
  __shared__ T as[kTile][kTile + 1], bs[kTile][kTile + 1];
  const int tx = threadIdx.x % kTile, ty = threadIdx.x / kTile;
  const int dt = I8 ? B2G_DTYPE_I8 : B2G_DTYPE_E4M3;
  const int64_t tn = (N + kTile - 1) / kTile, tiles = tn * ((M + kTile - 1) / kTile);
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t m0 = t / tn * kTile, n0 = t % tn * kTile;
    T acc = 0;
    for (int64_t k0 = 0; k0 < K; k0 += kTile) {
      as[ty][tx] = m0 + ty < M && k0 + tx < K ? (T)load_elem(A, (m0 + ty) * lda + k0 + tx, dt) : (T)0;
      bs[ty][tx] = n0 + ty < N && k0 + tx < K ? (T)load_elem(B, (n0 + ty) * ldb + k0 + tx, dt) : (T)0;
      __syncthreads();
      for (int k = 0; k < kTile; ++k) acc += as[ty][k] * bs[tx][k];
      __syncthreads();
    }
    const int64_t m = m0 + ty, n = n0 + tx;
    if (m < M && n < N) {
      float v = (float)acc;
      if (a_scale) v *= a_scale[m];
      if (b_scale) v *= b_scale[n];
      if (bias) v += bias[n];
      store_elem(C, m * ldc + n, c_dtype, v);
    }
  }
}

// dW tile by tile, tokens in ascending order.
__global__ void __launch_bounds__(kTile* kTile)
    wgrad_q8_generic_kernel(const void* dY, const void* Q, const float* scale, void* dW, int64_t M,
                            int64_t N, int64_t K, int64_t ldy, int64_t ldq, int64_t ldw, int dtype,
                            int q_dtype, bool accumulate, int c_dtype) {
  __shared__ float ys[kTile][kTile + 1], xs[kTile][kTile + 1];
  const int tx = threadIdx.x % kTile, ty = threadIdx.x / kTile;
  const int64_t tk = (K + kTile - 1) / kTile, tiles = tk * ((N + kTile - 1) / kTile);
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t n0 = t / tk * kTile, k0 = t % tk * kTile;
    float acc = 0.0f;
    for (int64_t m0 = 0; m0 < M; m0 += kTile) {
      const bool in = m0 + ty < M;
      ys[ty][tx] = in && n0 + tx < N ? load_elem(dY, (m0 + ty) * ldy + n0 + tx, dtype) : 0.0f;
      float x = 0.0f;
      if (in && k0 + tx < K) {
        x = load_elem(Q, (m0 + ty) * ldq + k0 + tx, q_dtype) * scale[m0 + ty];
        x = clamp_to(x, largest(dtype));
        x = dtype == B2G_DTYPE_BF16 ? __bfloat162float(__float2bfloat16_rn(x)) : __half2float(__float2half_rn(x));
      }
      xs[ty][tx] = x;
      __syncthreads();
      for (int m = 0; m < kTile; ++m) acc = fmaf(ys[m][ty], xs[m][tx], acc);
      __syncthreads();
    }
    const int64_t n = n0 + ty, k = k0 + tx;
    if (n < N && k < K) {
      if (accumulate) acc += static_cast<const float*>(dW)[n * ldw + k];
      store_elem(dW, n * ldw + k, c_dtype, acc);
    }
  }
}

unsigned tile_blocks(int64_t rows, int64_t cols, int sms) {
  const int64_t t = ((rows + kTile - 1) / kTile) * ((cols + kTile - 1) / kTile);
  return (unsigned)std::min<int64_t>(t, (int64_t)sms * 32);
}

}  // namespace
}  // namespace b2g

// ==================================================================== C ABI
using namespace b2g;

extern "C" int b2g_gemm_q8(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K,
                           int64_t lda, int64_t ldb, int64_t ldc, int dtype, const float* a_scale,
                           const float* b_scale, const float* bias, int c_dtype, void* stream) {
  clear_error();
  if (!is_q8(dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported 8-bit type code %d", dtype);
  if (!is_real(c_dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported output type code %d", c_dtype);
  if (M < 0 || N < 0 || K < 0) return fail(B2G_ERR_INVALID_ARG, "negative dimension");
  if (lda < std::max<int64_t>(K, 1) || ldb < std::max<int64_t>(K, 1) || ldc < std::max<int64_t>(N, 1))
    return fail(B2G_ERR_INVALID_ARG, "leading dimension smaller than the row length");
  if (dtype == B2G_DTYPE_I8 && K > 131071)
    return fail(B2G_ERR_INVALID_ARG, "int8 sums of K = %lld products can overflow int32 (at most 131071)",
                (long long)K);
  if (M == 0 || N == 0) {
    set_path(B2G_PATH_EMPTY);
    return B2G_OK;
  }
  if (!C) return fail(B2G_ERR_INVALID_ARG, "C is null");
  if (K > 0 && (!A || !B)) return fail(B2G_ERR_INVALID_ARG, "A or B is null");
  int dev = 0, sms = 0, cc = 0;
  int rc = current_device(&dev, &sms, &cc);
  if (rc != B2G_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned blocks = tile_blocks(M, N, sms);
  if (dtype == B2G_DTYPE_I8)
    gemm_q8_generic_kernel<true><<<blocks, kTile * kTile, 0, s>>>(A, B, C, M, N, K, lda, ldb, ldc, a_scale,
                                                                  b_scale, bias, c_dtype);
  else
    gemm_q8_generic_kernel<false><<<blocks, kTile * kTile, 0, s>>>(A, B, C, M, N, K, lda, ldb, ldc,
                                                                   a_scale, b_scale, bias, c_dtype);
  rc = launched("gemm_q8_generic_kernel");
  if (rc == B2G_OK) set_path(K == 0 ? B2G_PATH_ZERO : B2G_PATH_GENERIC);
  return rc;
}

extern "C" int b2g_wgrad_q8(const void* dY, const void* Q, const float* scale, void* dW, int64_t M,
                            int64_t N, int64_t K, int64_t ldy, int64_t ldq, int64_t ldw, int dtype,
                            int q_dtype, int accumulate, int c_dtype, void* stream) {
  clear_error();
  if (dtype != B2G_DTYPE_F16 && dtype != B2G_DTYPE_BF16)
    return fail(B2G_ERR_INVALID_ARG, "unsupported gradient type code %d", dtype);
  if (!is_q8(q_dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported 8-bit type code %d", q_dtype);
  if (!is_real(c_dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported output type code %d", c_dtype);
  if (accumulate && c_dtype != B2G_DTYPE_F32)
    return fail(B2G_ERR_INVALID_ARG, "a 16-bit dW is overwritten, not added to");
  if (M < 0 || N < 0 || K < 0) return fail(B2G_ERR_INVALID_ARG, "negative dimension");
  if (ldy < std::max<int64_t>(N, 1) || ldq < std::max<int64_t>(K, 1) || ldw < std::max<int64_t>(K, 1))
    return fail(B2G_ERR_INVALID_ARG, "leading dimension smaller than the row length");
  if (N == 0 || K == 0) {
    set_path(B2G_PATH_EMPTY);
    return B2G_OK;
  }
  if (!dW) return fail(B2G_ERR_INVALID_ARG, "dW is null");
  if (M > 0 && (!dY || !Q || !scale)) return fail(B2G_ERR_INVALID_ARG, "dY, Q or scale is null");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int dev = 0, sms = 0, cc = 0;
  int rc = current_device(&dev, &sms, &cc);
  if (rc != B2G_OK) return rc;
  wgrad_q8_generic_kernel<<<tile_blocks(N, K, sms), kTile * kTile, 0, s>>>(
      dY, Q, scale, dW, M, N, K, ldy, ldq, ldw, dtype, q_dtype, accumulate != 0, c_dtype);
  rc = launched("wgrad_q8_generic_kernel");
  if (rc == B2G_OK) set_path(M == 0 ? B2G_PATH_ZERO : B2G_PATH_GENERIC);
  return rc;
}
