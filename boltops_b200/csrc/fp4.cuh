// Microscaled 4-bit floating point: scales of a block, codes of eight values, and back.
//
// A code is e2m1 (0, .5, 1, 1.5, 2, 3, 4, 6 and a sign), two to a byte, the first in the low bits.
//   NV: blocks of 16, the scale an E4M3 byte: s = e4m3(min(amax * (1/6), 448)), code = e2m1(v / s)
//   MX: blocks of 32, the scale an E8M0 byte: the smallest 2^e with amax <= 6 * 2^e, 0 for a block
//       of zeros, code = e2m1(v / 2^e).  (The OCP MX specification's conversion, 2^(floor(log2 amax) - 2), is
//       half of that for amax between 6 and 8 times a power of two, and saturates there.)
// Codes are rounded to the nearest, ties to even, magnitudes above 6 to 6 (only NV has them: its
// scale may have been rounded down).  A block that holds a NaN or an infinity gets the NaN byte
// (0x7F, 0xFF) and codes 0.
#pragma once

#include <cuda_fp4.h>

#include "common.cuh"

namespace bolt {
namespace fp4 {

__device__ __forceinline__ bool finite_amax(float amax) {
  return __float_as_uint(amax) < 0x7F800000u;      // amax is not negative
}

// Scale byte of a block from its largest magnitude (a NaN or an infinity among the values must
// have made amax a NaN or an infinity).
template <bool NV>
__device__ __forceinline__ uint32_t scale_byte(float amax) {
  if (NV) {
    if (!finite_amax(amax)) return 0x7Fu;
    // (the product with the rounded 1/6 is exact wherever amax / 6 is the border of two E4M3 values:
    // 1/6 is rounded by 2^-25 of itself, half a step of any value by more)
    return __nv_cvt_float_to_fp8(amax * (float)(1.0 / 6.0), __NV_SATFINITE, __NV_E4M3);
  }
  if (!finite_amax(amax)) return 0xFFu;
  const uint32_t bits = __float_as_uint(amax);
  if (bits == 0) return 0u;
  // amax = 1.m * 2^(a - 127) <= 6 * 2^e = 1.5 * 2^(e + 2)
  const int byte = (int)(bits >> 23) - ((bits & 0x7FFFFFu) <= 0x400000u ? 2 : 1);
  return (uint32_t)max(byte, 0);
}

__device__ __forceinline__ float e4m3_to_f32(uint32_t byte) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3);
  return __half2float(__half(h));
}
__device__ __forceinline__ float e8m0_to_f32(uint32_t byte) {
  // 2^-127 is a denormal, 255 a NaN: both are the exponent bits with the fraction's highest bit set
  return __uint_as_float((byte << 23) | (((byte + 1) & 0xFFu) <= 1u ? 0x400000u : 0u));
}
template <bool NV>
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return NV ? e4m3_to_f32(byte) : e8m0_to_f32(byte);
}

// What a block's codes are made with: the scale and its reciprocal; 0 and 0 for codes 0.
struct Scaler {
  float s, r;
};
template <bool NV>
__device__ __forceinline__ Scaler scaler_of(uint32_t byte) {
  Scaler k;
  if (NV) {
    k.s = byte == 0x7Fu ? 0.f : e4m3_to_f32(byte);
    k.r = k.s > 0.f ? __frcp_rn(k.s) : 0.f;
  } else {
    k.s = 0.f;                                            // (not used: 1 / 2^e is exact)
    k.r = byte == 0xFFu ? 0.f : __uint_as_float((254u - byte) << 23);
    if (byte == 254u) k.r = __uint_as_float(0x400000u);
  }
  return k;
}

// v / s for the code.  MX: a product with a power of two, exact.  NV: the quotient q = v * r is
// corrected once by its remainder, which makes it the correctly rounded one (Markstein, "Computation
// of elementary functions on the IBM RISC System/6000 processor", 1990, with r the rounded
// reciprocal); rounded values of 16 bits lie on the border of two codes all the time, and v * r alone
// would decide such ties by the error of r.
template <bool NV>
__device__ __forceinline__ float quotient(float v, const Scaler& k) {
  const float q = v * k.r;
  if (!NV) return q;
  return fmaf(fmaf(-q, k.s, v), k.r, q);
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return (uint32_t)__nv_cvt_float2_to_fp4x2(make_float2(lo, hi), __NV_E2M1, cudaRoundNearest);
}
// eight values -> eight codes; k.r of 0 (a block of zeros or without finite values): codes 0
template <bool NV>
__device__ __forceinline__ uint32_t codes8(const float* v, const Scaler& k) {
  // (0 * infinity would be a NaN, and a NaN has no code: blocks with either have k.r = 0)
  if (k.r == 0.f) return 0u;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w |= pack2(quotient<NV>(v[2 * i], k), quotient<NV>(v[2 * i + 1], k)) << (8 * i);
  return w;
}

// |v| folded into a running maximum that a NaN passes through (fmaxf drops NaNs).
__device__ __forceinline__ float amax_nan(float m, float v) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(v)));
  return r;
}

// eight codes -> four packed pairs of halves (values 0 to 6, exact)
__device__ __forceinline__ void halves8(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n.reg .b8 b0, b1, b2, b3;\nmov.b32 {b0, b1, b2, b3}, %4;\n"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\ncvt.rn.f16x2.e2m1x2 %1, b1;\n"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\ncvt.rn.f16x2.e2m1x2 %3, b3;\n}\n"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}

}  // namespace fp4
}  // namespace bolt
