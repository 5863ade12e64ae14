// Row operators of the 8-bit linear layer: rows into 8 bits and out again, the RMS norm with an
// 8-bit output, and its backward pass.
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/b2g_gemm.h"
#include "errors.h"
#include "host.h"
#include "q8.cuh"

namespace b2g {
namespace {

using namespace q8;

constexpr int kRowThreads = 256;

// Sum (or integer maximum) over the block, returned to every thread.  `buf` holds one word per
// warp; the leading barrier lets consecutive calls share it.
__device__ __forceinline__ float block_sum(float v, float* buf) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.0f;
  for (int i = 0; i < (int)blockDim.x / 32; ++i) s += buf[i];
  return s;
}

__device__ __forceinline__ uint32_t block_max(uint32_t v, float* buf) {
  for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = __uint_as_float(v);
  __syncthreads();
  uint32_t s = 0;
  for (int i = 0; i < (int)blockDim.x / 32; ++i) s = max(s, __float_as_uint(buf[i]));
  return s;
}

struct NormArgs {
  const void *X, *R, *W;
  void *H, *Q;
  float *scale, *rstd;
  int64_t M, N, ldx, ldr, ldh, ldq;
  int dtype, w_dtype, q_dtype;
  float eps;
  bool norm, pow2;
};

// One block per row, two passes over it: sum of squares and largest |h * w| (|x| without the
// norm), then the 8-bit values.  The largest |y| is rstd * max|h * w|, so one pass serves both.
__global__ void __launch_bounds__(kRowThreads) rows_to_q8_kernel(const NormArgs a) {
  __shared__ float buf[kRowThreads / 32];
  for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x) {
    auto value = [&](int64_t n) {
      float h = load_elem(a.X, m * a.ldx + n, a.dtype);
      if (a.R) h += load_elem(a.R, m * a.ldr + n, a.dtype);
      return h;
    };
    float ss = 0.0f;
    uint32_t top = 0;
    for (int64_t n = threadIdx.x; n < a.N; n += blockDim.x) {
      const float h = value(n);
      const float v = a.norm ? h * load_elem(a.W, n, a.w_dtype) : h;
      ss = fmaf(h, h, ss);
      top = max(top, __float_as_uint(v) & 0x7fffffffu);
    }
    top = block_max(top, buf);
    float rstd = 1.0f;
    if (a.norm) rstd = 1.0f / sqrtf(block_sum(ss, buf) / (float)a.N + a.eps);
    const RowQuant rq = row_quant(top, rstd, q_max(a.q_dtype), a.pow2);
    if (threadIdx.x == 0) {
      a.scale[m] = rq.scale;
      if (a.rstd) a.rstd[m] = rstd;
    }
    const bool bad = rq.scale != rq.scale;
    for (int64_t n = threadIdx.x; n < a.N; n += blockDim.x) {
      const float h = value(n);
      const float v = a.norm ? h * load_elem(a.W, n, a.w_dtype) : h;
      static_cast<uint8_t*>(a.Q)[m * a.ldq + n] = bad ? 0 : (uint8_t)to_q8(quotient(v, rq), a.q_dtype);
      if (a.H) store_elem(a.H, m * a.ldh + n, a.dtype, h);
    }
  }
}

__global__ void __launch_bounds__(kRowThreads)
    dequantize_kernel(const void* Q, const float* scale, void* X, int64_t M, int64_t N, int64_t ldq,
                      int64_t ldx, int q_dtype, int dtype) {
  for (int64_t m = blockIdx.x; m < M; m += gridDim.x) {
    const float s = scale[m];
    for (int64_t n = threadIdx.x; n < N; n += blockDim.x) {
      store_elem(X, m * ldx + n, dtype, clamp_to(load_elem(Q, m * ldq + n, q_dtype) * s, largest(dtype)));
    }
  }
}

struct BwdArgs {
  const void *dY, *X, *W, *dR;
  const float *x_scale, *rstd;
  void* dX;
  float* part;  // [blocks][N] partial sums of dw, or null
  int64_t M, N, ldy, ldx, ldr, lddx;
  int dtype, x_dtype, w_dtype;
};

// One block per row: mean(g * xh), then dx.
__global__ void __launch_bounds__(kRowThreads) rmsnorm_bwd_kernel(const BwdArgs a) {
  __shared__ float buf[kRowThreads / 32];
  for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x) {
    const float rstd = a.rstd[m];
    const float xs = a.x_scale ? a.x_scale[m] : 1.0f;
    float c = 0.0f;
    for (int64_t n = threadIdx.x; n < a.N; n += blockDim.x) {
      const float xh = load_elem(a.X, m * a.ldx + n, a.x_dtype) * xs * rstd;
      c = fmaf(load_elem(a.dY, m * a.ldy + n, a.dtype) * load_elem(a.W, n, a.w_dtype), xh, c);
    }
    c = block_sum(c, buf) / (float)a.N;
    for (int64_t n = threadIdx.x; n < a.N; n += blockDim.x) {
      const float xh = load_elem(a.X, m * a.ldx + n, a.x_dtype) * xs * rstd;
      const float dy = load_elem(a.dY, m * a.ldy + n, a.dtype);
      float dx = rstd * (dy * load_elem(a.W, n, a.w_dtype) - xh * c);
      if (a.dR) dx += load_elem(a.dR, m * a.ldr + n, a.dtype);
      if (a.part) {
        float* p = a.part + (int64_t)blockIdx.x * a.N + n;
        *p = (m == blockIdx.x ? 0.0f : *p) + dy * xh;
      }
      store_elem(a.dX, m * a.lddx + n, a.dtype, dx);
    }
  }
}

// dw[n] = sum over the blocks' partial sums, in block order.
__global__ void __launch_bounds__(kRowThreads)
    dw_sum_kernel(const float* part, float* dw, int64_t N, int blocks) {
  const int64_t n = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (n >= N) return;
  float s = 0.0f;
  for (int b = 0; b < blocks; ++b) s += part[(int64_t)b * N + n];
  dw[n] = s;
}


unsigned row_blocks(int64_t M, int sms) { return (unsigned)std::min<int64_t>(M, (int64_t)sms * 8); }

// Checks that every row operator shares: extents and leading dimensions.
int check_rows(int64_t M, int64_t N, std::initializer_list<int64_t> lds) {
  if (M < 0 || N < 0) return fail(B2G_ERR_INVALID_ARG, "negative dimension");
  for (int64_t ld : lds)
    if (ld < std::max<int64_t>(N, 1))
      return fail(B2G_ERR_INVALID_ARG, "leading dimension smaller than the row length");
  return B2G_OK;
}

int rows_to_q8(const NormArgs& a, cudaStream_t s) {
  int dev = 0, sms = 0, cc = 0;
  const int rc = current_device(&dev, &sms, &cc);
  if (rc != B2G_OK) return rc;
  rows_to_q8_kernel<<<row_blocks(a.M, sms), kRowThreads, 0, s>>>(a);
  return launched("rows_to_q8_kernel");
}

}  // namespace

int dequantize_rows(const void* Q, const float* scale, void* X, int64_t M, int64_t N, int64_t ldq,
                    int64_t ldx, int q_dtype, int dtype, cudaStream_t s) {
  int dev = 0, sms = 0, cc = 0;
  const int rc = current_device(&dev, &sms, &cc);
  if (rc != B2G_OK) return rc;
  dequantize_kernel<<<row_blocks(M, sms), kRowThreads, 0, s>>>(Q, scale, X, M, N, ldq, ldx, q_dtype,
                                                               dtype);
  return launched("dequantize_kernel");
}

}  // namespace b2g

// ==================================================================== C ABI
using namespace b2g;

extern "C" int b2g_quantize_q8(const void* X, void* Q, float* scale, int64_t M, int64_t N,
                               int64_t ldx, int64_t ldq, int dtype, int q_dtype, int pow2,
                               void* stream) {
  clear_error();
  if (!is_real(dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported input type code %d", dtype);
  if (!is_q8(q_dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported 8-bit type code %d", q_dtype);
  const int rc = check_rows(M, N, {ldx, ldq});
  if (rc != B2G_OK) return rc;
  if (M == 0) return B2G_OK;
  if (N == 0) return fail(B2G_ERR_INVALID_ARG, "rows of no elements have no scale");
  if (!X || !Q || !scale) return fail(B2G_ERR_INVALID_ARG, "X, Q or scale is null");
  NormArgs a{};
  a.X = X;
  a.Q = Q;
  a.scale = scale;
  a.M = M; a.N = N; a.ldx = ldx; a.ldq = ldq;
  a.dtype = dtype; a.w_dtype = dtype; a.q_dtype = q_dtype;
  a.pow2 = pow2 != 0;
  return rows_to_q8(a, static_cast<cudaStream_t>(stream));
}

extern "C" int b2g_dequantize_q8(const void* Q, const float* scale, void* X, int64_t M, int64_t N,
                                 int64_t ldq, int64_t ldx, int q_dtype, int dtype, void* stream) {
  clear_error();
  if (!is_real(dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported output type code %d", dtype);
  if (!is_q8(q_dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported 8-bit type code %d", q_dtype);
  const int rc = check_rows(M, N, {ldx, ldq});
  if (rc != B2G_OK) return rc;
  if (M == 0 || N == 0) return B2G_OK;
  if (!X || !Q || !scale) return fail(B2G_ERR_INVALID_ARG, "X, Q or scale is null");
  return dequantize_rows(Q, scale, X, M, N, ldq, ldx, q_dtype, dtype,
                         static_cast<cudaStream_t>(stream));
}

extern "C" int b2g_rmsnorm_q8(const void* X, const void* R, const void* W, void* H, void* Q,
                              float* scale, float* rstd, int64_t M, int64_t N, int64_t ldx,
                              int64_t ldr, int64_t ldh, int64_t ldq, int dtype, int w_dtype,
                              int q_dtype, float eps, int pow2, void* stream) {
  clear_error();
  if (!is_real(dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported input type code %d", dtype);
  if (!is_real(w_dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported weight type code %d", w_dtype);
  if (!is_q8(q_dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported 8-bit type code %d", q_dtype);
  const int rc = check_rows(M, N, {ldx, R ? ldr : ldx, H ? ldh : ldx, ldq});
  if (rc != B2G_OK) return rc;
  if (!(eps >= 0.0f)) return fail(B2G_ERR_INVALID_ARG, "eps is negative or NaN");
  if (M == 0) return B2G_OK;
  if (N == 0) return fail(B2G_ERR_INVALID_ARG, "rows of no elements have no norm");
  if (!X || !W || !Q || !scale) return fail(B2G_ERR_INVALID_ARG, "X, W, Q or scale is null");
  if (H && ((H == X && ldh != ldx) || (H == R && ldh != ldr)))
    return fail(B2G_ERR_INVALID_ARG, "H in place needs the leading dimension of what it replaces");
  NormArgs a{};
  a.X = X; a.R = R; a.W = W; a.H = H; a.Q = Q;
  a.scale = scale; a.rstd = rstd;
  a.M = M; a.N = N; a.ldx = ldx; a.ldr = ldr; a.ldh = ldh; a.ldq = ldq;
  a.dtype = dtype; a.w_dtype = w_dtype; a.q_dtype = q_dtype;
  a.eps = eps;
  a.norm = true;
  a.pow2 = pow2 != 0;
  return rows_to_q8(a, static_cast<cudaStream_t>(stream));
}

extern "C" int b2g_rmsnorm_bwd_q8(const void* dY, const void* X, const float* x_scale, const void* W,
                                  const float* rstd, const void* dR, void* dX, float* dw, int64_t M,
                                  int64_t N, int64_t ldy, int64_t ldx, int64_t ldr, int64_t lddx,
                                  int dtype, int x_dtype, int w_dtype, void* stream) {
  clear_error();
  if (!is_real(dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported gradient type code %d", dtype);
  if (!is_real(w_dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported weight type code %d", w_dtype);
  if (!is_real(x_dtype) && !is_q8(x_dtype))
    return fail(B2G_ERR_INVALID_ARG, "unsupported checkpoint type code %d", x_dtype);
  int rc = check_rows(M, N, {ldy, ldx, dR ? ldr : ldy, lddx});
  if (rc != B2G_OK) return rc;
  if (N == 0) return B2G_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (M == 0) {  // no token: dw is a sum of nothing
    if (!dw) return B2G_OK;
    const cudaError_t e = cudaMemsetAsync(dw, 0, (size_t)N * sizeof(float), s);
    return e == cudaSuccess ? B2G_OK : cuda_fail(e, "cudaMemsetAsync(dw)");
  }
  if (!dY || !X || !W || !rstd || !dX)
    return fail(B2G_ERR_INVALID_ARG, "dY, X, W, rstd or dX is null");
  if (is_q8(x_dtype) != (x_scale != nullptr))
    return fail(B2G_ERR_INVALID_ARG, "x_scale goes with an 8-bit checkpoint, and only with one");
  if ((dX == dY && lddx != ldy) || (dX == dR && lddx != ldr))
    return fail(B2G_ERR_INVALID_ARG, "dX in place needs the leading dimension of what it replaces");
  int dev = 0, sms = 0, cc = 0;
  rc = current_device(&dev, &sms, &cc);
  if (rc != B2G_OK) return rc;
  BwdArgs a{};
  a.dY = dY; a.X = X; a.W = W; a.dR = dR;
  a.x_scale = x_scale; a.rstd = rstd;
  a.dX = dX;
  a.M = M; a.N = N; a.ldy = ldy; a.ldx = ldx; a.ldr = ldr; a.lddx = lddx;
  a.dtype = dtype; a.x_dtype = x_dtype; a.w_dtype = w_dtype;
  const unsigned blocks = row_blocks(M, sms);
  Workspace ws(s);
  if (dw) {
    rc = ws.alloc((size_t)blocks * (size_t)N * sizeof(float), "cudaMallocFromPoolAsync(dw partial sums)");
    if (rc != B2G_OK) return rc;
    a.part = static_cast<float*>(ws.get());
  }
  rmsnorm_bwd_kernel<<<blocks, kRowThreads, 0, s>>>(a);
  rc = launched("rmsnorm_bwd_kernel");
  if (rc != B2G_OK || !dw) return rc;
  dw_sum_kernel<<<(unsigned)((N + kRowThreads - 1) / kRowThreads), kRowThreads, 0, s>>>(
      a.part, dw, N, (int)blocks);
  return launched("dw_sum_kernel");
}
