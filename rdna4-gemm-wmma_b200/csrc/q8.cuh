// Device helpers of the 8-bit operators: element conversion and the rounding of a row to 8 bits.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "../../include/b2g_gemm.h"

namespace b2g {
namespace q8 {

// Element i of an array of type `dt` (B2G_DTYPE_*) as fp32, exact for every type.
__device__ __forceinline__ float load_elem(const void* base, int64_t i, int dt) {
  switch (dt) {
    case B2G_DTYPE_F16: return __half2float(static_cast<const __half*>(base)[i]);
    case B2G_DTYPE_BF16: return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
    case B2G_DTYPE_F32: return static_cast<const float*>(base)[i];
    case B2G_DTYPE_I8: return (float)static_cast<const int8_t*>(base)[i];
    default: return float(static_cast<const __nv_fp8_e4m3*>(base)[i]);
  }
}

// Store v, rounded to nearest even once, as element i of an array of type `dt` (F16, BF16, F32).
__device__ __forceinline__ void store_elem(void* base, int64_t i, int dt, float v) {
  switch (dt) {
    case B2G_DTYPE_F16: static_cast<__half*>(base)[i] = __float2half_rn(v); break;
    case B2G_DTYPE_BF16: static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v); break;
    default: static_cast<float*>(base)[i] = v; break;
  }
}

// Largest finite value of a type, and v clamped to it (NaN stays).  A row's largest value may round
// to one 8-bit step above it, which would pass the type's range at its very end.
__device__ __forceinline__ float largest(int dt) {
  return dt == B2G_DTYPE_F16 ? 65504.0f : __uint_as_float(dt == B2G_DTYPE_BF16 ? 0x7f7f0000u : 0x7f7fffffu);
}
__device__ __forceinline__ float clamp_to(float v, float top) {
  return v > top ? top : v < -top ? -top : v;
}

// How the elements v of a row become 8-bit values t.  v is first scaled by a power of two that brings
// the row's largest value near 1 (exact, and no later product overflows); then
//   without pow2   t = v * qmax / amax, the quotient correctly rounded: for 16-bit v it often lies
//                  exactly on the border between two 8-bit values (amax / 2 is 63.5 int8 steps), and
//                  a product with a rounded reciprocal would fall to either side of it.  v * qmax is
//                  exact for such v (11 + 7 significant bits); the quotient is one Newton correction
//                  of the product with rcp, which is correctly rounded when rcp is (P. Markstein,
//                  1990);
//   pow2, or a scale at its floor   t = v / scale, exact for the norm's factor 1 (den = 0).
struct RowQuant {
  float mul, den, rcp;
  float scale;  // NaN for a row that holds a NaN or an infinity (its 8-bit values are 0)
};

constexpr float kMinScale = 1.17549435e-38f;  // 2^-126: the reciprocal of every scale is finite

__device__ __forceinline__ float q_max(int q_dtype) { return q_dtype == B2G_DTYPE_I8 ? 127.0f : 448.0f; }

// amax_bits: bits of the largest |v| of the row, compared as integers, so that NaN and
// infinity win.  The row's values are v * factor (1, or the norm's rstd).
__device__ __forceinline__ RowQuant row_quant(uint32_t amax_bits, float factor, float qmax, bool pow2) {
  RowQuant r;
  const float top = __uint_as_float(amax_bits);
  const float amax = top * factor;
  if (amax_bits >= 0x7f800000u || !(amax < __int_as_float(0x7f800000))) {
    r.mul = r.den = r.rcp = 0.0f;
    r.scale = __int_as_float(0x7fc00000);
    return r;
  }
  float s = amax / qmax;
  if (s < kMinScale) s = kMinScale;
  if (pow2) {
    const uint32_t b = __float_as_uint(s);  // a normal number: round up to the next power of two
    s = __uint_as_float((b + 0x007fffffu) & 0x7f800000u);
  }
  r.scale = s;
  // 2^-k with 2^k the binade of top, at most 2^100 (a zero or subnormal top)
  const int k = max((int)(amax_bits >> 23) - 127, -100);
  const float p = k < 127 ? __uint_as_float((uint32_t)(127 - k) << 23) : 0x1p-127f;
  if (pow2 || s == kMinScale) {
    r.mul = p;
    r.den = 0.0f;
    r.rcp = factor / (s * p);
  } else {
    r.mul = qmax * p;
    r.den = top * p;
    r.rcp = 1.0f / r.den;
  }
  return r;
}

__device__ __forceinline__ float quotient(float v, const RowQuant& r) {
  const float a = v * r.mul;
  const float t = a * r.rcp;
  return r.den == 0.0f ? t : fmaf(fmaf(-t, r.den, a), r.rcp, t);
}

// t rounded to nearest even as one byte of type q_dtype.  |t| <= qmax by construction.
__device__ __forceinline__ uint32_t to_q8(float t, int q_dtype) {
  if (q_dtype == B2G_DTYPE_I8) return (uint32_t)__float2int_rn(t) & 0xffu;
  return (uint32_t)__nv_cvt_float_to_fp8(t, __NV_SATFINITE, __NV_E4M3);
}

// N values v of a row as 8-bit bytes (zeros for a bad row).
template <int N>
__device__ __forceinline__ void pack_q8(const float (&v)[N], const RowQuant& r, int q_dtype, bool bad,
                                        uint8_t (&o)[N]) {
  if constexpr (N % 4 == 0) {
    uint32_t* w = reinterpret_cast<uint32_t*>(o);
    float t[N];
    if (r.den == 0.0f) {
#pragma unroll
      for (int j = 0; j < N; ++j) t[j] = v[j] * r.mul * r.rcp;
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) t[j] = quotient(v[j], r);
    }
    if (q_dtype == B2G_DTYPE_I8) {
      // 1.5 * 2^23 added: the sum's unit is 1, so the addition rounds t to an integer (to nearest
      // even) and leaves its two's complement in the low byte
#pragma unroll
      for (int j = 0; j < N; j += 4) {
        const uint32_t a = __float_as_uint(t[j] + 12582912.0f), b = __float_as_uint(t[j + 1] + 12582912.0f);
        const uint32_t c = __float_as_uint(t[j + 2] + 12582912.0f), d = __float_as_uint(t[j + 3] + 12582912.0f);
        w[j / 4] = __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; j += 4) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(t[j], t[j + 1]), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(t[j + 2], t[j + 3]), __NV_SATFINITE, __NV_E4M3);
        w[j / 4] = lo | hi << 16;
      }
    }
    if (bad) {
#pragma unroll
      for (int j = 0; j < N / 4; ++j) w[j] = 0;
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = bad ? 0 : (uint8_t)to_q8(quotient(v[j], r), q_dtype);
  }
}

}  // namespace q8
}  // namespace b2g
