// fp4_format.cuh -- the microscaled 4-bit formats.
//
// Values are E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two to a byte, the even
// column in the low nibble.  Each block of consecutive columns of a row has one scale byte:
//   LMOE_FP4_MX  blocks of 32, E8M0 scales 2^(byte - 127), byte 255 = NaN
//                byte = clamp(floor(log2 max|x|) - 2, -127, 127) + 127
//   LMOE_FP4_NV  blocks of 16, E4M3 scales under an fp32 tensor scale g
//                s = E4M3(max|x| / (6 g)), at most 448
// and a value is code(x / scale) * scale, rounded to the nearest code (ties to even), at most 6.
// A block that holds an infinity or a NaN gets the NaN scale and zero codes.
// Scale rows are padded to a multiple of 32 bytes, so that the product reads whole sectors.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "lmoe_b200.h"

namespace lmoe {

__host__ __device__ constexpr int fp4_block(int format) { return format == LMOE_FP4_NV ? 16 : 32; }
__host__ __device__ constexpr int fp4_scale_pitch(int K, int format) { return (K / fp4_block(format) + 31) / 32 * 32; }

// Eight values -> eight codes (the first in the lowest nibble): round to nearest even, at most 6.
__device__ __forceinline__ uint32_t fp4_pack8(const float* v) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

__device__ __forceinline__ float e8m0_value(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7fc00000u)
                      : (byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23));
}
__device__ __forceinline__ float e4m3_value(uint32_t byte) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
}

// 1 / x, off by at most one unit in the last place (2^-23).
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Scale byte of an MX block whose largest absolute value is amax (finite).  *mul = 1 / scale: a
// power of two, so x / scale is exact.
__device__ __forceinline__ uint32_t fp4_mx_scale(float amax, float* mul) {
  int e = (int)(__float_as_uint(amax) >> 23) - 127 - 2;   // below the normal range: the clamp applies either way
  e = e < -127 ? -127 : e;
  *mul = __uint_as_float((uint32_t)(127 - e) << 23);      // 2^-e, -125 <= -e <= 127
  return (uint32_t)(e + 127);
}

// NV: s is the E4M3 value nearest to amax / (6 g), at most 448.
// Exactly: the double quotient cannot land on the wrong side of a midpoint, since amax and
// midpoint * 6 g are integers of at most 31 bits in a common unit and differ by more than 2^-32
// relative or not at all.
static __device__ __noinline__ float fp4_nv_scale_exact(float amax, float g) {
  const double t = (double)amax / (6.0 * (double)g);
  if (t >= 448.0) return 448.0f;
  const float tf = (float)t;
  int e = (int)(__float_as_uint(tf) >> 23) - 127;
  e = e < -6 ? -6 : e;
  // a quotient just below a power of two may round up to it in fp32: the step is then twice the
  // true one, but the nearest value is the power of two itself either way
  const double step = (double)__uint_as_float((uint32_t)(e - 3 + 127) << 23);
  const double inv = (double)__uint_as_float((uint32_t)(3 - e + 127) << 23);
  return (float)(rint(t * inv) * step);
}
// r6 = rcp_approx(6 g): the product with it is off by less than 2^-22 + 2^-24, below 2^-17 of a
// step (a value has at most 16), so clear of a midpoint by 2^-16 its rounding is the exact one.  Near
// a midpoint (16-bit values meet it exactly about once in 30 blocks) the sign of midpoint * 6 g - amax
// decides: midpoint * 6 has 8 bits, and the fused multiply-add keeps the sign of what is left.
__device__ __forceinline__ float fp4_nv_scale(float amax, float g, float r6) {
  const float t = __fmul_rn(amax, r6);
  int e = (int)(__float_as_uint(t) >> 23) - 127;
  e = e < -6 ? -6 : e;
  const float u = __fmul_rn(t, __uint_as_float((uint32_t)(3 - e + 127) << 23));   // exact, in steps
  float n = rintf(u);
  if (!(t < 440.0f) || !(t > 1e-30f) || !(amax > 1e-20f)) return amax > 0.0f ? fp4_nv_scale_exact(amax, g) : 0.0f;
  const float step = __uint_as_float((uint32_t)(e - 3 + 127) << 23);
  const float low = floorf(u);
  if (fabsf(u - low - 0.5f) < 0x1p-16f) {
    const float over = __fmaf_rn(__fmul_rn(__fmul_rn(low + 0.5f, step), 6.0f), g, -amax);   // of the midpoint
    n = over > 0.0f ? low : (over < 0.0f ? low + 1.0f : 2.0f * rintf(0.5f * low + 0.25f));
  }
  return __fmul_rn(n, step);
}

// Code of |x| by exact comparisons with the borders b * s * g between codes: b * s is exact in
// fp32 and the fused multiply-add keeps the sign of (b * s) * g - |x| (small values are scaled up,
// so that the difference does not fall below the smallest fp32).
__device__ __forceinline__ uint32_t fp4_exact_code(float x, float s, float g) {
  const float up = fabsf(x) < 0x1p-80f ? 0x1p64f : 1.0f;
  const float ax = fabsf(x) * up;
  s *= up;
  uint32_t c = 0;
  c += __fmaf_rn(0.25f * s, g, -ax) < 0.0f;    // ties go to the even code: > or >= in turn
  c += __fmaf_rn(0.75f * s, g, -ax) <= 0.0f;
  c += __fmaf_rn(1.25f * s, g, -ax) < 0.0f;
  c += __fmaf_rn(1.75f * s, g, -ax) <= 0.0f;
  c += __fmaf_rn(2.5f * s, g, -ax) < 0.0f;
  c += __fmaf_rn(3.5f * s, g, -ax) <= 0.0f;
  c += __fmaf_rn(5.0f * s, g, -ax) < 0.0f;
  return c | (__float_as_uint(x) >> 31 << 3);
}

// Codes of 16 values of at most 11 significant bits under a scale d of at most four, r = rcp_approx(d).
// They may meet a border between codes exactly, and one that is missed is missed by 2^-12 (11 bits
// against 7).  The quotient is corrected by its exact remainder: a quotient that is a border comes out
// as that border (the remainder is a few units of q times d, which fp32 holds, and the correction is
// off by 2^-23 of them), and the conversion takes the even code.  No value may be above 8 d: where a
// quotient overflows, its correction would be the difference of two infinities.
__device__ __forceinline__ uint2 fp4_short_codes(const float* a, float d, float r) {
  float q[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float q0 = __fmul_rn(a[i], -r);   // of the quotient's opposite: then zeros keep their signs
    q[i] = __fmaf_rn(-__fmaf_rn(q0, d, a[i]), r, q0);
  }
  return make_uint2(fp4_pack8(q) ^ 0x88888888u, fp4_pack8(q + 8) ^ 0x88888888u);
}

// The codes come from the rounded product with the reciprocal (three roundings and the reciprocal's
// unit, below 2^-21 relative); where a border lies that near, they come from fp4_exact_code.
//
// SHORT: the values are 16-bit.  Under a g that is a power of two they meet borders in nearly every
// warp, and take fp4_short_codes at once (32768 x 4096 bf16 values, g = 1: 75 us; with the comparisons
// in every such warp 195).  Not so blocks with values beyond 8 d, under a scale at its limit of 448:
// their products saturate with the right sign (cutting the values at 8 d instead cost every block: 97 us
// against 84 in one run).
template <bool SHORT>
__device__ __forceinline__ uint32_t fp4_encode_nv(const float* a, float amax, float g, float r6, uint2& codes) {
  const float s = fp4_nv_scale(amax, g, r6);
  codes = make_uint2(0u, 0u);
  if (s > 0.0f) {
    const float d = __fmul_rn(s, g);
    const bool plain = d > 1e-30f && d < 1e30f;
    const float r = rcp_approx(plain ? d : 1.0f);
    const bool corrected = plain && (__float_as_uint(g) & 0x7fffffu) == 0 && amax <= __fmul_rn(8.0f, d);
    if (SHORT && corrected) {
      codes = fp4_short_codes(a, d, r);
      return (uint32_t)__nv_cvt_float_to_fp8(s, __NV_SATFINITE, __NV_E4M3);
    }
    float lo[16], hi[16];
    const float down = 1.0f - 0x1p-20f, upf = 1.0f + 0x1p-20f;
    const float rl = __fmul_rn(r, down), rh = __fmul_rn(r, upf);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      lo[i] = __fmul_rn(a[i], rl);
      hi[i] = __fmul_rn(a[i], rh);
    }
    codes.x = fp4_pack8(lo);
    codes.y = fp4_pack8(lo + 8);
    if (!plain || codes.x != fp4_pack8(hi) || codes.y != fp4_pack8(hi + 8)) {
      uint32_t low = 0;   // bits that 16-bit values, widened to fp32, do not have
#pragma unroll
      for (int i = 0; i < 16; ++i) low |= __float_as_uint(a[i]) & 0x1fffu;
      if (corrected && low == 0) {
        codes = fp4_short_codes(a, d, r);
      } else {
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i >> 3] |= fp4_exact_code(a[i], s, g) << (4 * (i & 7));
        codes = make_uint2(w[0], w[1]);
      }
    }
  }
  return (uint32_t)__nv_cvt_float_to_fp8(s, __NV_SATFINITE, __NV_E4M3);
}

}  // namespace lmoe
