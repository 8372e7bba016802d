// fp4_quant.cu -- rows to the microscaled 4-bit formats (fp4_format.cuh) and back.
//
// Quantising reads 2 (or 4) bytes a value and writes 1/2 byte and 1/32 or 1/16 of a scale byte:
// memory bound, if few instructions are spent on a value: a thread owns 32 consecutive values (two
// 32-byte loads of 16-bit values; one MX block, two NV blocks) so that what a thread costs is
// spread over them (with 16 values a thread: 217 instructions a warp for 512 values, and bound by
// their issue at 4.8 TB/s).  The maximum is taken on the absolute values' bit patterns, which
// order like the values and put infinities and NaN on top.  With `positions` each row is
// written to several output rows, so that a MoE layer's permutation costs no pass of its own:
// the row is quantised once and the copies are 4-bit.
//
// 32768 x 4096 values: MX bf16 52 us (6.6 TB/s), fp32 99 us (6.2); NV fp32 101 us (6.1); NV bf16 75 us
// (4.6 TB/s), bound by the issue of its instructions (the quotients' corrections, fp4_format.cuh).
#include <cuda_bf16.h>

#include "fp4_format.cuh"
#include "host_util.h"
#include "ptx.cuh"

namespace lmoe {
namespace {

struct QuantArgs {
  const void* x;
  int64_t ldx;               // elements between rows
  int64_t rows;
  int K, format;
  const float* global_scale;
  int64_t rows_per_scale;    // rows under one tensor scale (NV)
  const int32_t* positions;  // [rows, copies] output rows, or NULL: row r goes to row r
  int copies;
  int64_t out_rows;
  uint8_t* q;
  uint8_t* scales;
  int64_t pitch;             // bytes between scale rows
  int vec;                   // rows of x start at multiples of 32 or 16 bytes (0: neither)
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

// The bits of 32 consecutive values.
template <typename T>
__device__ __forceinline__ void load32(const T* p, int vec, uint32_t (&w)[8 * sizeof(T)]) {
  constexpr int kWords = 8 * (int)sizeof(T);
  if (vec == 32) {
#pragma unroll
    for (int i = 0; i < kWords / 8; ++i) {
      uint32_t v[8];
      ld_global_nc_v8(reinterpret_cast<const uint32_t*>(p) + 8 * i, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[8 * i + j] = v[j];
    }
  } else if (vec == 16) {
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + i);
      w[4 * i] = u.x;
      w[4 * i + 1] = u.y;
      w[4 * i + 2] = u.z;
      w[4 * i + 3] = u.w;
    }
  } else {
    T* e = reinterpret_cast<T*>(w);
#pragma unroll
    for (int i = 0; i < 32; ++i) e[i] = p[i];
  }
}
// Sixteen of them as fp32, and the largest bit pattern of their absolute values.
__device__ __forceinline__ uint32_t widen16(const uint32_t* w, const float*, float* a) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    a[i] = __uint_as_float(w[i]);
    top = max(top, w[i] & 0x7fffffffu);
  }
  return top;
}
template <typename T>
__device__ __forceinline__ uint32_t widen16(const uint32_t* w, const T*, float* a) {
  // 16-bit patterns order like the values too: two maxima at a time, widened at the end
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  const uint16_t h = (uint16_t)max(m & 0xffffu, m >> 16);
#pragma unroll
  for (int i = 0; i < 16; ++i) a[i] = to_float<T>(reinterpret_cast<const T*>(w)[i]);
  return __float_as_uint(to_float<T>(*reinterpret_cast<const T*>(&h)));
}

// blockDim = (chunks of 32 columns, rows); grid.x walks the chunks of the padded scale row,
// grid.y the rows.
template <typename T, int FORMAT>
__global__ void __launch_bounds__(256) quantize_fp4_kernel(const QuantArgs a) {
  constexpr bool kMx = FORMAT == LMOE_FP4_MX;
  const int chunk = blockIdx.x * blockDim.x + threadIdx.x;
  if (chunk * (kMx ? 1 : 2) >= (int)a.pitch) return;
  const bool ok = chunk < a.K / 32;   // else: padding of the scale row
  for (int64_t r = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; r < a.rows; r += (int64_t)gridDim.y * blockDim.y) {
    uint2 codes[2] = {make_uint2(0u, 0u), make_uint2(0u, 0u)};
    uint32_t scale[2] = {0u, 0u};
    if (ok) {
      uint32_t w[8 * sizeof(T)];
      load32<T>(static_cast<const T*>(a.x) + r * a.ldx + (int64_t)chunk * 32, a.vec, w);
      float v[32];
      const uint32_t t0 = widen16(w, static_cast<const T*>(nullptr), v);
      const uint32_t t1 = widen16(w + 4 * sizeof(T), static_cast<const T*>(nullptr), v + 16);
      constexpr uint32_t kInf = 0x7f800000u;
      if (kMx) {
        const uint32_t top = max(t0, t1);
        scale[0] = 255u;
        if (top < kInf) {
          float mul;
          scale[0] = fp4_mx_scale(__uint_as_float(top), &mul);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __fmul_rn(v[i], mul);
          codes[0] = make_uint2(fp4_pack8(v), fp4_pack8(v + 8));
          codes[1] = make_uint2(fp4_pack8(v + 16), fp4_pack8(v + 24));
        }
      } else {
        const float g = a.global_scale ? __ldg(a.global_scale + (a.rows_per_scale >= a.rows ? 0 : r / a.rows_per_scale))
                                       : 1.0f;
        const bool fine = g > 0.0f && g < __uint_as_float(kInf);
        const float r6 = rcp_approx(__fmul_rn(6.0f, g));
        scale[0] = fine && t0 < kInf ? fp4_encode_nv<sizeof(T) == 2>(v, __uint_as_float(t0), g, r6, codes[0]) : 0x7fu;
        scale[1] = fine && t1 < kInf ? fp4_encode_nv<sizeof(T) == 2>(v + 16, __uint_as_float(t1), g, r6, codes[1]) : 0x7fu;
      }
    }
    for (int j = 0; j < a.copies; ++j) {
      const int64_t o = a.positions ? (int64_t)__ldg(a.positions + r * a.copies + j) : r;
      if (o < 0 || o >= a.out_rows) continue;
      if (ok)
        *reinterpret_cast<uint4*>(a.q + o * (a.K / 2) + (int64_t)chunk * 16) =
            make_uint4(codes[0].x, codes[0].y, codes[1].x, codes[1].y);
      uint8_t* sp = a.scales + o * a.pitch;
      if (kMx)
        sp[chunk] = (uint8_t)scale[0];
      else
        reinterpret_cast<uint16_t*>(sp)[chunk] = (uint16_t)(scale[0] | scale[1] << 8);
    }
  }
}

template <int FORMAT>
__global__ void __launch_bounds__(256)
    dequantize_fp4_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scales, int64_t pitch,
                          int64_t rows, int K, const float* __restrict__ global_scale, int64_t rows_per_scale,
                          __nv_bfloat16* __restrict__ out) {
  const bool vec32 = (reinterpret_cast<uintptr_t>(out) & 31) == 0;   // K % 32 == 0: then every chunk
  const int chunk = blockIdx.x * blockDim.x + threadIdx.x;
  if (chunk >= K / 32) return;
  for (int64_t r = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; r < rows; r += (int64_t)gridDim.y * blockDim.y) {
    const uint4 c = __ldg(reinterpret_cast<const uint4*>(q + r * (K / 2) + (int64_t)chunk * 16));
    const uint8_t* sp = scales + r * pitch;
    const float g = FORMAT == LMOE_FP4_NV && global_scale
                        ? __ldg(global_scale + (rows_per_scale >= rows ? 0 : r / rows_per_scale)) : 1.0f;
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    __nv_bfloat16* dst = out + r * K + (int64_t)chunk * 32;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float s = FORMAT == LMOE_FP4_MX ? e8m0_value(sp[chunk]) : e4m3_value(sp[2 * chunk + h]);
      uint32_t o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t h2;
        asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b0;\n\t}"
            : "=r"(h2)
            : "r"(w[2 * h + (i >> 2)] >> (8 * (i & 3))));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
        // code * scale is exact in fp32; the tensor scale and bf16 round once each
        float x = __fmul_rn(f.x, s), y = __fmul_rn(f.y, s);
        if (FORMAT == LMOE_FP4_NV) {
          x = __fmul_rn(x, g);
          y = __fmul_rn(y, g);
        }
        const __nv_bfloat162 p = __floats2bfloat162_rn(x, y);
        o[i] = *reinterpret_cast<const uint32_t*>(&p);
      }
      if (vec32) {
        st_global_v8(dst + 16 * h, o);
      } else {
        reinterpret_cast<uint4*>(dst + 16 * h)[0] = make_uint4(o[0], o[1], o[2], o[3]);
        reinterpret_cast<uint4*>(dst + 16 * h)[1] = make_uint4(o[4], o[5], o[6], o[7]);
      }
    }
  }
}

struct RowGrid {
  dim3 grid, block;
};

RowGrid row_grid(int chunks, int64_t rows) {
  const int bx = chunks >= 256 ? 256 : (chunks + 31) / 32 * 32;
  const int by = 256 / bx;
  const int64_t gy = (rows + by - 1) / by;
  RowGrid g;
  g.block = dim3((unsigned)bx, (unsigned)by);
  g.grid = dim3((unsigned)((chunks + bx - 1) / bx), (unsigned)(gy < 32768 ? gy : 32768));
  return g;
}

template <typename T>
void launch_quantize(const QuantArgs& a, cudaStream_t stream) {
  // chunks of the padded scale row: the threads behind the last column zero its padding
  const int chunks = (int)(a.pitch * fp4_block(a.format) / 32);
  const RowGrid g = row_grid(chunks, a.rows);
  if (a.format == LMOE_FP4_MX)
    quantize_fp4_kernel<T, LMOE_FP4_MX><<<g.grid, g.block, 0, stream>>>(a);
  else
    quantize_fp4_kernel<T, LMOE_FP4_NV><<<g.grid, g.block, 0, stream>>>(a);
}

}  // namespace
}  // namespace lmoe

using namespace lmoe;

extern "C" int lmoe_fp4_scale_pitch(int K, int format) {
  LMOE_ARG_CHECK(format == LMOE_FP4_MX || format == LMOE_FP4_NV);
  LMOE_ARG_CHECK(K > 0 && K % 32 == 0);
  return fp4_scale_pitch(K, format);
}

extern "C" int lmoe_quantize_fp4(const void* x, int dtype, int64_t rows, int K, int64_t ldx, int format,
                                 const float* global_scale, int64_t rows_per_scale, const int32_t* positions,
                                 int copies, int64_t out_rows, uint8_t* q, uint8_t* scales, lmoe_stream_t stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  LMOE_ARG_CHECK(dtype == LMOE_DTYPE_BF16 || dtype == LMOE_DTYPE_F16 || dtype == LMOE_DTYPE_F32);
  LMOE_ARG_CHECK(format == LMOE_FP4_MX || format == LMOE_FP4_NV);
  LMOE_ARG_CHECK(rows >= 0 && K > 0 && K % 32 == 0 && ldx >= K && out_rows >= 0);
  LMOE_ARG_CHECK(positions ? copies >= 1 : (copies == 1 && out_rows == rows));
  LMOE_ARG_CHECK(!global_scale || rows_per_scale >= 1);
  if (rows == 0) return LMOE_OK;
  LMOE_ARG_CHECK(x && q && scales && aligned16(q) && (reinterpret_cast<uintptr_t>(scales) & 1) == 0);
  const int64_t esize = dtype == LMOE_DTYPE_F32 ? 4 : 2;
  LMOE_ARG_CHECK(reinterpret_cast<uintptr_t>(x) % esize == 0);
  QuantArgs a;
  a.x = x;
  a.ldx = ldx;
  a.rows = rows;
  a.K = K;
  a.format = format;
  a.global_scale = global_scale;
  a.rows_per_scale = global_scale ? rows_per_scale : 1;
  a.positions = positions;
  a.copies = copies;
  a.out_rows = out_rows;
  a.q = q;
  a.scales = scales;
  a.pitch = fp4_scale_pitch(K, format);
  const uintptr_t at = reinterpret_cast<uintptr_t>(x) | (uintptr_t)(ldx * esize);
  a.vec = at % 32 == 0 ? 32 : (at % 16 == 0 ? 16 : 0);
  if (dtype == LMOE_DTYPE_BF16)
    launch_quantize<__nv_bfloat16>(a, stream);
  else if (dtype == LMOE_DTYPE_F16)
    launch_quantize<__half>(a, stream);
  else
    launch_quantize<float>(a, stream);
  return cuda_status(cudaGetLastError());
}

extern "C" int lmoe_dequantize_fp4(const uint8_t* q, const uint8_t* scales, int64_t scale_pitch, int64_t rows, int K,
                                   int format, const float* global_scale, int64_t rows_per_scale, void* out,
                                   lmoe_stream_t stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  LMOE_ARG_CHECK(format == LMOE_FP4_MX || format == LMOE_FP4_NV);
  LMOE_ARG_CHECK(rows >= 0 && K > 0 && K % 32 == 0 && scale_pitch >= K / fp4_block(format));
  LMOE_ARG_CHECK(!global_scale || rows_per_scale >= 1);
  if (rows == 0) return LMOE_OK;
  LMOE_ARG_CHECK(q && scales && out && aligned16(out) && aligned16(q));
  const RowGrid g = row_grid(K / 32, rows);
  const int64_t rps = global_scale ? rows_per_scale : 1;
  if (format == LMOE_FP4_MX)
    dequantize_fp4_kernel<LMOE_FP4_MX><<<g.grid, g.block, 0, stream>>>(q, scales, scale_pitch, rows, K, global_scale,
                                                                      rps, static_cast<__nv_bfloat16*>(out));
  else
    dequantize_fp4_kernel<LMOE_FP4_NV><<<g.grid, g.block, 0, stream>>>(q, scales, scale_pitch, rows, K, global_scale,
                                                                      rps, static_cast<__nv_bfloat16*>(out));
  return cuda_status(cudaGetLastError());
}
