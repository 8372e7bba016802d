// fp8_format.cuh -- 8-bit floating point (E4M3) with one fp32 scale per block of 128 columns.
//
//   s = max(max|x| / 448, 2^-126)    over 128 columns of a row, or over 128 x 128 of a matrix
//       (optionally rounded up to a power of two);  NaN where the block holds an infinity or NaN
//   code = x / s to the nearest E4M3 value, ties to even (0 in a block that is not finite)
//
// The quotient's rounding is exact.  A reciprocal times x is within 2^-22 of the quotient, so its
// products with a reciprocal 2^-21 too small and one 2^-21 too large enclose it, and where both
// round to the same code that is the code; where they differ (a few values in 10^5) the quotient
// is divided and corrected by its remainder.  Two multiplications and one two-value conversion a
// value cost less than a division.
#pragma once
#include <cstdint>
#include <cuda_fp16.h>

namespace lmoe {

constexpr int kFp8Block = 128;
constexpr float kFp8Top = 448.0f;

__device__ __forceinline__ uint16_t cvt_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t cvt_e4m3x4(float a, float b, float c, float d) {
  return (uint32_t)cvt_e4m3x2(a, b) | (uint32_t)cvt_e4m3x2(c, d) << 16;
}
// Values of the two low bytes / the two high bytes of w (exact in fp16).
__device__ __forceinline__ uint32_t e4m3x2_half2(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_half2_high(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(w));
  return r;
}

// Scale of a block from the bits of its largest absolute value; NaN unless that is finite.
__device__ __forceinline__ float fp8_scale(uint32_t top, bool power_of_two) {
  if (top >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
  float s = fmaxf(__fdiv_rn(__uint_as_float(top), kFp8Top), __uint_as_float(0x00800000u));
  // s is normal and below 2^120: the next power of two is a carry out of the fraction
  if (power_of_two) s = __uint_as_float((__float_as_uint(s) + 0x007fffffu) & 0x7f800000u);
  return s;
}

// x / s rounded to odd: the value that a later rounding to fewer bits cannot tell from the quotient.
__device__ __forceinline__ float fp8_exact_quotient(float x, float s) {
  if (s < __uint_as_float(0x21800000u)) {   // 2^-60: keeps the remainder above the subnormals
    x *= __uint_as_float(0x67800000u);      // 2^80, exact for what such a block holds
    s *= __uint_as_float(0x67800000u);
  }
  const float q = __fdiv_rn(x, s);
  const float rem = __fmaf_rn(-q, s, x);
  const uint32_t b = __float_as_uint(q);
  if (rem == 0.0f || (b & 1u)) return q;
  return __uint_as_float((rem < 0.0f) == (x < 0.0f) ? b + 1u : b - 1u);   // (q may be a zero, whose rem is x)
}

// The reciprocals that enclose 1 / s.
struct Fp8Inverse {
  float s, lo, hi;
  __device__ __forceinline__ explicit Fp8Inverse(float scale) : s(scale) {
    const float r = __frcp_rn(scale);
    const bool power = (__float_as_uint(scale) & 0x007fffffu) == 0;   // then the products are exact
    lo = power ? r : __fmul_rn(r, 1.0f - 0x1p-21f);
    hi = power ? r : __fmul_rn(r, 1.0f + 0x1p-21f);
  }
};

// Codes of four values, the first in the lowest byte.
__device__ __forceinline__ uint32_t fp8_encode4(const float* x, const Fp8Inverse& v) {
  const uint32_t a = cvt_e4m3x4(__fmul_rn(x[0], v.lo), __fmul_rn(x[1], v.lo), __fmul_rn(x[2], v.lo),
                                __fmul_rn(x[3], v.lo));
  const uint32_t b = cvt_e4m3x4(__fmul_rn(x[0], v.hi), __fmul_rn(x[1], v.hi), __fmul_rn(x[2], v.hi),
                                __fmul_rn(x[3], v.hi));
  if (a == b) return a;
  return cvt_e4m3x4(fp8_exact_quotient(x[0], v.s), fp8_exact_quotient(x[1], v.s), fp8_exact_quotient(x[2], v.s),
                    fp8_exact_quotient(x[3], v.s));
}

}  // namespace lmoe
