// fp4_quant.cu -- rows to the microscaled 4-bit formats (fp4_format.cuh) and back.
//
// Quantising reads 2 (or 4) bytes a value and writes 1/2 byte and 1/32 or 1/16 of a scale byte:
// memory bound.  A thread owns 16 consecutive values (one 32-byte load of 16-bit values), an MX
// block is two neighbouring lanes; the maximum is taken on the absolute values' bit patterns,
// which order like the values and put infinities and NaN on top.  With `positions` each row is
// written to several output rows, so that a MoE layer's permutation costs no pass of its own:
// the row is quantised once and the copies are 4-bit.
#include <cuda_bf16.h>

#include "fp4_format.cuh"
#include "host_util.h"

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
  int vec;                   // rows of x start at multiples of 16 bytes
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float(float v) { return v; }

template <typename T>
__device__ __forceinline__ void load16(const T* p, bool vec, float (&a)[16]) {
  if (vec) {
    constexpr int kPieces = 16 * (int)sizeof(T) / 16, kPer = 16 / (int)sizeof(T);
    uint4 u[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) u[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const T* e = reinterpret_cast<const T*>(&u[i]);
#pragma unroll
      for (int j = 0; j < kPer; ++j) a[i * kPer + j] = to_float<T>(e[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) a[i] = to_float<T>(p[i]);
  }
}

// blockDim = (chunks of 16 columns, rows); grid.x walks the chunks of the padded scale row,
// grid.y the rows.
template <typename T, int FORMAT>
__global__ void __launch_bounds__(256) quantize_fp4_kernel(const QuantArgs a) {
  const int chunk = blockIdx.x * blockDim.x + threadIdx.x;
  const int chunks = a.K / 16;
  const int nscale = a.K / fp4_block(FORMAT);
  for (int64_t r = (int64_t)blockIdx.y * blockDim.y + threadIdx.y;; r += (int64_t)gridDim.y * blockDim.y) {
    const bool row_ok = r < a.rows;
    if (!__any_sync(0xffffffffu, row_ok)) break;
    const bool ok = row_ok && chunk < chunks;
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = 0.0f;
    if (ok) load16<T>(static_cast<const T*>(a.x) + r * a.ldx + (int64_t)chunk * 16, a.vec != 0, v);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    if (FORMAT == LMOE_FP4_MX) top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    if (!row_ok) continue;
    uint2 codes = make_uint2(0u, 0u);
    uint32_t scale = 0;
    if (ok) {
      const float g = FORMAT == LMOE_FP4_NV && a.global_scale ? __ldg(a.global_scale + (a.rows_per_scale >= a.rows ? 0 : r / a.rows_per_scale)) : 1.0f;
      const bool fine = top < 0x7f800000u && g > 0.0f && g < __uint_as_float(0x7f800000u);
      if (!fine)
        scale = FORMAT == LMOE_FP4_MX ? 255u : 0x7fu;
      else if (FORMAT == LMOE_FP4_MX)
        scale = fp4_encode_mx(v, __uint_as_float(top), codes);
      else
        scale = fp4_encode_nv(v, __uint_as_float(top), g, codes);
    }
    // MX: the even lane of a block stores its scale; padding behind the last scale is zero
    const int sc = FORMAT == LMOE_FP4_MX ? chunk >> 1 : chunk;
    const bool store_scale = (FORMAT == LMOE_FP4_NV || (chunk & 1) == 0) && sc < (int)a.pitch;
    if (sc >= nscale) scale = 0;
    for (int j = 0; j < a.copies; ++j) {
      const int64_t o = a.positions ? (int64_t)__ldg(a.positions + r * a.copies + j) : r;
      if (o < 0 || o >= a.out_rows) continue;
      if (ok) *reinterpret_cast<uint2*>(a.q + o * (a.K / 2) + (int64_t)chunk * 8) = codes;
      if (store_scale) a.scales[o * a.pitch + sc] = (uint8_t)scale;
    }
  }
}

template <int FORMAT>
__global__ void __launch_bounds__(256)
    dequantize_fp4_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scales, int64_t pitch,
                          int64_t rows, int K, const float* __restrict__ global_scale, int64_t rows_per_scale,
                          __nv_bfloat16* __restrict__ out) {
  const int chunk = blockIdx.x * blockDim.x + threadIdx.x;
  if (chunk >= K / 16) return;
  for (int64_t r = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; r < rows; r += (int64_t)gridDim.y * blockDim.y) {
    const uint2 c = __ldg(reinterpret_cast<const uint2*>(q + r * (K / 2) + (int64_t)chunk * 8));
    const uint32_t sb = scales[r * pitch + (FORMAT == LMOE_FP4_MX ? chunk >> 1 : chunk)];
    const float s = FORMAT == LMOE_FP4_MX ? e8m0_value(sb) : e4m3_value(sb);
    const float g = FORMAT == LMOE_FP4_NV && global_scale ? __ldg(global_scale + (rows_per_scale >= rows ? 0 : r / rows_per_scale)) : 1.0f;
    const uint32_t w[2] = {c.x, c.y};
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t b = (w[i >> 2] >> (8 * (i & 3))) & 0xffu;
      uint32_t h2;
      asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b0;\n\t}"
          : "=r"(h2)
          : "r"(b));
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
      // code * scale is exact in fp32; the tensor scale and bf16 round once each
      const __nv_bfloat162 p = __floats2bfloat162_rn(__fmul_rn(__fmul_rn(f.x, s), g), __fmul_rn(__fmul_rn(f.y, s), g));
      o[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
    uint4* dst = reinterpret_cast<uint4*>(out + r * K + (int64_t)chunk * 16);
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
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
  const int chunks = (int)a.pitch * fp4_block(a.format) / 16;
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
  LMOE_ARG_CHECK(x && q && scales && (reinterpret_cast<uintptr_t>(q) & 7) == 0);
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
  a.vec = aligned16(x) && (ldx * esize) % 16 == 0;
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
  LMOE_ARG_CHECK(q && scales && out && aligned16(out) && (reinterpret_cast<uintptr_t>(q) & 7) == 0);
  const RowGrid g = row_grid(K / 16, rows);
  const int64_t rps = global_scale ? rows_per_scale : 1;
  if (format == LMOE_FP4_MX)
    dequantize_fp4_kernel<LMOE_FP4_MX><<<g.grid, g.block, 0, stream>>>(q, scales, scale_pitch, rows, K, global_scale,
                                                                      rps, static_cast<__nv_bfloat16*>(out));
  else
    dequantize_fp4_kernel<LMOE_FP4_NV><<<g.grid, g.block, 0, stream>>>(q, scales, scale_pitch, rows, K, global_scale,
                                                                      rps, static_cast<__nv_bfloat16*>(out));
  return cuda_status(cudaGetLastError());
}
