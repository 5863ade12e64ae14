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

// Two fp32 values in one register pair: sm_100 multiplies, adds and fuses pairs in one instruction,
// which matters where a row kernel's instructions, not its bytes, are the limit.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_get(F2 x, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v));
}
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
// max(top, |v|), NaN if either is (so that a row's largest value tells of every NaN in it).
__device__ __forceinline__ float max_abs(float top, float v) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(top), "f"(fabsf(v)));
  return r;
}

// Four 8-bit values of a word as fp32 pairs.  int8: the byte with its sign bit flipped, placed in the low
// byte of 2^23, is 2^23 + 128 + value (a conversion instruction runs at an eighth of this rate).
__device__ __forceinline__ void unpack_q8x4(uint32_t w, int q_dtype, F2& lo, F2& hi) {
  if (q_dtype == B2G_DTYPE_I8) {
    w ^= 0x80808080u;
    const F2 off = f2(-8388736.0f, -8388736.0f);
    lo = f2_add(f2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440)),
                   __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441))), off);
    hi = f2_add(f2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7442)),
                   __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7443))), off);
  } else {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a));
    const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&b));
    lo = f2(x.x, x.y);
    hi = f2(y.x, y.y);
  }
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

// N values v of a row as 8-bit values, one in the low byte of each word (zeros for a bad row).
template <int N>
__device__ __forceinline__ void round_q8(const float (&v)[N], const RowQuant& r, int q_dtype, bool bad,
                                         uint32_t (&o)[N]) {
  static_assert(N % 2 == 0, "pairs");
  const F2 mul = f2(r.mul, r.mul), rcp = f2(r.rcp, r.rcp), nden = f2(-r.den, -r.den);
  F2 t[N / 2];
  if (r.den == 0.0f) {
#pragma unroll
    for (int j = 0; j < N / 2; ++j) t[j] = f2_mul(f2_mul(f2(v[2 * j], v[2 * j + 1]), mul), rcp);
  } else {
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {  // quotient(), two at a time
      const F2 a = f2_mul(f2(v[2 * j], v[2 * j + 1]), mul);
      const F2 q = f2_mul(a, rcp);
      t[j] = f2_fma(f2_fma(q, nden, a), rcp, q);
    }
  }
  if (q_dtype == B2G_DTYPE_I8) {
    // 1.5 * 2^23 added: the sum's unit is 1, so the addition rounds t to an integer (to nearest
    // even) and leaves its two's complement in the low byte
    const F2 magic = f2(12582912.0f, 12582912.0f);
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      float a, b;
      f2_get(f2_add(t[j], magic), a, b);
      o[2 * j] = __float_as_uint(a);
      o[2 * j + 1] = __float_as_uint(b);
    }
  } else {
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      float a, b;
      f2_get(t[j], a, b);
      o[2 * j] = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
      o[2 * j + 1] = o[2 * j] >> 8;
    }
  }
  if (bad) {
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = 0;
  }
}

// The same as packed bytes.
template <int N>
__device__ __forceinline__ void pack_q8(const float (&v)[N], const RowQuant& r, int q_dtype, bool bad,
                                        uint8_t (&o)[N]) {
  if constexpr (N % 4 == 0) {
    uint32_t b[N];
    round_q8<N>(v, r, q_dtype, bad, b);
    uint32_t* w = reinterpret_cast<uint32_t*>(o);
#pragma unroll
    for (int j = 0; j < N / 4; ++j)
      w[j] = __byte_perm(__byte_perm(b[4 * j], b[4 * j + 1], 0x0040),
                         __byte_perm(b[4 * j + 2], b[4 * j + 3], 0x0040), 0x5410);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = bad ? 0 : (uint8_t)to_q8(quotient(v[j], r), q_dtype);
  }
}

}  // namespace q8
}  // namespace b2g
