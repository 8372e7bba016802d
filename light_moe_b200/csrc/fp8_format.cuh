// fp8_format.cuh -- 8-bit floating point (E4M3) with one fp32 scale per block of 128 columns.
//
//   s = max(max|x| / 448, 2^-126)    over 128 columns of a row, or over 128 x 128 of a matrix
//       (optionally rounded up to a power of two);  NaN where the block holds an infinity or NaN
//   code = x / s to the nearest E4M3 value, ties to even (0 in a block that is not finite)
//
// The quotient's rounding is exact.  A reciprocal times x is within 2^-22 of the quotient, so its
// products with a reciprocal 2^-21 too small and one 2^-21 too large enclose it, and where both
// round to the same code that is the code.  Where they differ, by one step, x is compared with the
// midpoint times s, whose difference a fused multiply-add gives exactly.  That is no rare case: 3/4 of a
// block's largest value (and 3/8, 3/16 ...) is such a midpoint, 336 of 448, and one in 128 of 16-bit values;
// with a division there, 32768 x 4096 bf16 values took 170 us instead of 121, and as below, without
// any comparison, 78 (71 with one row a thread in flight).
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

// For values of at most 11 significant bits no comparison is needed.  Where s = rn(max / 448) is no power of two, a
// value x and a midpoint m (5 bits) either have 448 x = m max, or differ by more than 2^-16, integers of at most 16
// bits; then s, which is within 2^-24 of max / 448, does not change their order.  Where they are equal, x / s lies
// above m (in size) if 448 s < max, below if 448 s > max, and is m if they are equal: the same for the whole block.
// So a reciprocal that is 2^-17 too large, too small or neither, and products rounded to 18 bits (midpoints stay, and
// what is 2^-16 away stays on its side), give the code.  With a power of two the products are exact.
__device__ __forceinline__ float fp8_inverse16(float scale, float top) {
  const float r = __frcp_rn(scale), rest = __fmaf_rn(-kFp8Top, scale, top);   // (exact)
  if ((__float_as_uint(scale) & 0x007fffffu) == 0 || rest == 0.0f) return r;
  return __fmul_rn(r, rest > 0.0f ? 1.0f + 0x1p-17f : 1.0f - 0x1p-17f);
}

// Codes of four values times r, the first in the lowest byte (two products to an instruction).
template <bool SNAP = false>
__device__ __forceinline__ uint32_t fp8_scaled4(const float* x, float r) {
  float p[4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\tmul.rn.f32x2 a, a, b;\n\t"
        "mov.b64 {%0, %1}, a;\n\t}"
        : "=f"(p[2 * i]), "=f"(p[2 * i + 1])
        : "f"(x[2 * i]), "f"(x[2 * i + 1]), "f"(r));
  if constexpr (SNAP)   // 18 significant bits
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = __uint_as_float((__float_as_uint(p[i]) + 0x20u) & ~0x3fu);
  return cvt_e4m3x4(p[0], p[1], p[2], p[3]);
}

// Codes of four values from those below (lo) and above, with one of the two for each.
static __device__ __noinline__ uint32_t fp8_between4(uint32_t lo, uint32_t hi, float x0, float x1, float x2, float x3,
                                                     float s) {
  if (s < __uint_as_float(0x21800000u)) {   // 2^-60: the difference must not end below the subnormals
    const float up = __uint_as_float(0x67800000u);   // 2^80, exact for what such a block holds
    x0 *= up;
    x1 *= up;
    x2 *= up;
    x3 *= up;
    s *= up;
  }
  const float x[4] = {x0, x1, x2, x3};
  uint32_t step = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t l2 = h ? e4m3x2_half2_high(lo) : e4m3x2_half2(lo), h2 = h ? e4m3x2_half2_high(hi) : e4m3x2_half2(hi);
    const float2 l = __half22float2(*reinterpret_cast<const __half2*>(&l2));
    const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&h2));
    const float mid[2] = {0.5f * (l.x + u.x), 0.5f * (l.y + u.y)};   // exact: five bits (of equal codes: no matter)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = 2 * h + i;
      const float rest = __fmaf_rn(-mid[i], s, x[at]);   // (twice x may be infinite)
      const bool beyond = rest != 0.0f ? (rest < 0.0f) == (x[at] < 0.0f) : (lo >> (8 * at) & 1u) != 0u;   // ties to even
      if (beyond) step |= 0xffu << (8 * at);
    }
  }
  return (lo & ~step) | (hi & step);
}
__device__ __forceinline__ uint4 fp8_encode16(const float (&x)[16], const Fp8Inverse& v) {
  uint32_t a[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] = fp8_scaled4(x + 4 * i, v.lo);
    const uint32_t b = fp8_scaled4(x + 4 * i, v.hi);
    if (a[i] != b) a[i] = fp8_between4(a[i], b, x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3], v.s);
  }
  return make_uint4(a[0], a[1], a[2], a[3]);
}
// Of values of 16-bit types; r from fp8_inverse16.
__device__ __forceinline__ uint4 fp8_encode16(const float (&x)[16], float r) {
  return make_uint4(fp8_scaled4<true>(x, r), fp8_scaled4<true>(x + 4, r), fp8_scaled4<true>(x + 8, r),
                    fp8_scaled4<true>(x + 12, r));
}

}  // namespace lmoe
