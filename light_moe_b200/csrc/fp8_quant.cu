// fp8_quant.cu -- values to 8-bit floating point with a scale per block of 128 (fp8_format.cuh) and back.
//
// Rows: a thread owns 16 consecutive values and eight threads a block of 128 columns, whose largest
// absolute value they find with three shuffles on the bit patterns (which order like the values
// and put infinities and NaN on top).  Matrices: a CTA holds a block of 128 x 128 in registers, so
// that the values are read once.  Row scales are stored block after block ([K blocks][rows], rows padded
// to four): the product reads a block's scales of 128 rows at a time.
//
// Matrices are bound by HBM (64 x 1408 x 2048 fp32 there and back 304 us, 1.85 GB: 6.1 TB/s), and so
// are large calls of rows (32768 x 4096 bf16: 71 us, 5.7 TB/s; fp32 115, 5.9 TB/s; 8192 rows bf16 22).  Back, 8192 x 4096
// to bf16: 16-20 us.  Matrices of 16-bit values, 64 x 1408 x 2048: 119 us, 4.7 TB/s: half the bytes for the same barriers and codes.
#include <cuda_bf16.h>

#include <type_traits>

#include "fp8_format.cuh"
#include "host_util.h"
#include "ptx.cuh"

namespace lmoe {
namespace {

struct Fp8RowArgs {
  const void* x;
  int64_t ldx;               // elements between rows
  int64_t rows;
  int K;
  int power_of_two;
  const int32_t* positions;  // [rows, copies] output rows, or NULL: row r goes to row r
  int copies;
  int64_t out_rows;
  uint8_t* q;
  float* scales;
  int64_t pitch;             // elements between the scales of neighbouring K blocks
  int vec;                   // rows of x start at multiples of 32 or 16 bytes (0: neither)
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float(float v) { return v; }

// The bits of 16 consecutive values.
template <typename T>
__device__ __forceinline__ void load16(const T* p, int vec, uint32_t (&w)[4 * sizeof(T)]) {
  constexpr int kWords = 4 * (int)sizeof(T);
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
    for (int i = 0; i < 16; ++i) e[i] = p[i];
  }
}
// Bits, as fp32, of the largest absolute value of 16.
template <typename T>
__device__ __forceinline__ uint32_t top16(const uint32_t (&w)[4 * sizeof(T)]) {
  uint32_t m = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, w[i] & 0x7fffffffu);
    return m;
  } else {
    // 16-bit patterns order like the values too: two maxima at a time, widened at the end
#pragma unroll
    for (int i = 0; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
    const uint16_t h = (uint16_t)max(m & 0xffffu, m >> 16);
    return __float_as_uint(to_float<T>(*reinterpret_cast<const T*>(&h)));
  }
}
template <typename T>
__device__ __forceinline__ uint4 encode16(const uint32_t (&w)[4 * sizeof(T)], float s, uint32_t top) {
  if (!(s == s)) return make_uint4(0u, 0u, 0u, 0u);
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = to_float<T>(reinterpret_cast<const T*>(w)[i]);
  if constexpr (sizeof(T) == 2)
    return fp8_encode16(v, fp8_inverse16(s, __uint_as_float(top)));
  else
    return fp8_encode16(v, Fp8Inverse(s));
}

// blockDim = (chunks of 16 * kParts columns, a multiple of 32; rows); grid.x walks the chunks, grid.y the rows.
// Of 16-bit values a thread takes 32 of a row, which spreads a block's scale, its reciprocal and the addresses (32768 x
// 4096 bf16: 86 us with 16), and one row at a time (72 us, with two 80); of fp32 16 of two rows, whose loads are in flight
// together (115 us, with one row 117).
template <typename T>
constexpr int kParts = sizeof(T) == 2 ? 2 : 1;
template <typename T>
constexpr int kRows = sizeof(T) == 2 ? 1 : 2;
template <typename T>
__global__ void __launch_bounds__(256) quantize_fp8_rows_kernel(const Fp8RowArgs a) {
  constexpr int P = kParts<T>, R = kRows<T>, kLanes = 8 / P;   // of a block
  const int chunk = blockIdx.x * blockDim.x + threadIdx.x, col = chunk * 16 * P;
  const int64_t stride = (int64_t)gridDim.y * blockDim.y;
  const T* x = static_cast<const T*>(a.x) + col;
  for (int64_t r0 = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; r0 < a.rows; r0 += R * stride) {
    uint32_t w[R][P][4 * sizeof(T)];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (col + 16 * p < a.K && r0 + i * stride < a.rows)
          load16<T>(x + (r0 + i * stride) * a.ldx + 16 * p, a.vec, w[i][p]);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t r = r0 + i * stride;
      if (r >= a.rows) break;
      uint32_t top = 0u;
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (col + 16 * p < a.K) top = max(top, top16<T>(w[i][p]));
      // all 32 lanes are of one row, kLanes of one block
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (col >= a.K) continue;
      const float s = fp8_scale(top, a.power_of_two != 0);
      uint4 codes[P];
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (col + 16 * p < a.K) codes[p] = encode16<T>(w[i][p], s, top);
      for (int j = 0; j < a.copies; ++j) {
        const int64_t o = a.positions ? (int64_t)__ldg(a.positions + r * a.copies + j) : r;
        if (o < 0 || o >= a.out_rows) continue;
#pragma unroll
        for (int p = 0; p < P; ++p)
          if (col + 16 * p < a.K) *reinterpret_cast<uint4*>(a.q + o * a.K + col + 16 * p) = codes[p];
        if ((chunk & (kLanes - 1)) == 0) a.scales[(int64_t)(chunk / kLanes) * a.pitch + o] = s;
      }
    }
  }
}

// One CTA a block of 128 x 128: thread t owns 16 columns (t % 8) of the rows t / 8 and 64 + t / 8.
constexpr int kBlockThreads = 512;
template <typename T>
__global__ void __launch_bounds__(kBlockThreads)
    quantize_fp8_blocks_kernel(const T* __restrict__ x, int64_t rows, int K, int vec, int power_of_two,
                               uint8_t* __restrict__ q, float* __restrict__ scales, int row_blocks, int kblocks,
                               int64_t total) {
  __shared__ uint32_t part[2][kBlockThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int buf = 0;
  for (int64_t b = blockIdx.x; b < total; b += gridDim.x, buf ^= 1) {
    const int kb = (int)(b % kblocks);
    const int64_t rb = b / kblocks;   // over all matrices
    const int64_t mat = rb / row_blocks, r0 = (rb % row_blocks) * kFp8Block;
    const int c = kb * kFp8Block + (tid & 7) * 16;
    uint32_t w[2][4 * sizeof(T)], top = 0;
    bool ok[2];
    int64_t at[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t r = r0 + (tid >> 3) + 64 * i;
      ok[i] = r < rows && c < K;
      at[i] = (mat * rows + r) * K + c;
      if (ok[i]) load16<T>(x + at[i], vec, w[i]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (ok[i]) top = max(top, top16<T>(w[i]));
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) part[buf][warp] = top;
    __syncthreads();   // the other buffer's readers are behind the next one
    top = part[buf][lane & (kBlockThreads / 32 - 1)];
#pragma unroll
    for (int o = 1; o < kBlockThreads / 32; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float s = fp8_scale(top, power_of_two != 0);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (ok[i]) *reinterpret_cast<uint4*>(q + at[i]) = encode16<T>(w[i], s, top);
    if (tid == 0) scales[b] = s;
  }
}

struct Fp8ScaleStrides {
  int64_t mat, row, block;   // elements between matrices, row blocks and K blocks
};

template <typename T>
__device__ __forceinline__ void store16(T* dst, const float (&v)[16], bool vec32) {
  constexpr int kWords = 4 * (int)sizeof(T);
  uint32_t w[kWords];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kWords / 8; ++i) {
    uint32_t o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = w[8 * i + j];
    if (vec32) {
      st_global_v8(reinterpret_cast<uint32_t*>(dst) + 8 * i, o);
    } else {
      reinterpret_cast<uint4*>(dst)[2 * i] = make_uint4(o[0], o[1], o[2], o[3]);
      reinterpret_cast<uint4*>(dst)[2 * i + 1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
    dequantize_fp8_kernel(const uint8_t* __restrict__ q, const float* __restrict__ scales, Fp8ScaleStrides st,
                          int64_t rows, int64_t total_rows, int K, int block_shift, T* __restrict__ out) {
  constexpr int kAhead = 4;   // rows whose loads are in flight
  const bool vec32 = (reinterpret_cast<uintptr_t>(out) & 31) == 0;   // K % 16 == 0: then every chunk
  const int chunk = blockIdx.x * blockDim.x + threadIdx.x;
  if (chunk >= K / 16) return;
  const int64_t stride = (int64_t)gridDim.y * blockDim.y;
  for (int64_t r0 = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; r0 < total_rows; r0 += kAhead * stride) {
    uint4 c[kAhead];
    float s[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t r = r0 + i * stride;
      if (r >= total_rows) break;
      c[i] = __ldg(reinterpret_cast<const uint4*>(q + r * K + (int64_t)chunk * 16));
      const int64_t mat = rows == total_rows ? 0 : r / rows, in = r - mat * rows;
      s[i] = __ldg(scales + mat * st.mat + (in >> block_shift) * st.row + (int64_t)(chunk >> 3) * st.block);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t r = r0 + i * stride;
      if (r >= total_rows) break;
      const uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
      float v[16];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = e4m3x2_half2(w[j]), hi = e4m3x2_half2_high(w[j]);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        v[4 * j] = __fmul_rn(a.x, s[i]);
        v[4 * j + 1] = __fmul_rn(a.y, s[i]);
        v[4 * j + 2] = __fmul_rn(b.x, s[i]);
        v[4 * j + 3] = __fmul_rn(b.y, s[i]);
      }
      store16<T>(out + r * K + (int64_t)chunk * 16, v, vec32);
    }
  }
}

// Column indexes are counted in 32 bits, up to the end of a CTA's last chunks (256 threads of 32 columns).
constexpr int kMaxColumns = INT32_MAX - 256 * 32;

struct RowGrid {
  dim3 grid, block;
};

// CTAs for all SMs to hold a few at a time, no more than there are rows for.
RowGrid row_grid(int chunks, int64_t rows, int sms) {
  const int bx = chunks >= 256 ? 256 : (chunks + 31) / 32 * 32;
  const int by = 256 / bx;
  const int64_t gx = (chunks + bx - 1) / bx, gy = (rows + by - 1) / by;
  const int64_t most = (8 * (int64_t)sms + gx - 1) / gx;
  RowGrid g;
  g.block = dim3((unsigned)bx, (unsigned)by);
  g.grid = dim3((unsigned)gx, (unsigned)(gy < most ? gy : most));
  return g;
}

int vector_bytes(const void* x, int64_t pitch_bytes) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(x) | (uintptr_t)pitch_bytes;
  return at % 32 == 0 ? 32 : (at % 16 == 0 ? 16 : 0);
}

template <typename T>
void launch_blocks(const void* x, int64_t rows, int K, int vec, int power, uint8_t* q, float* scales, int64_t count,
                   int sms, cudaStream_t stream) {
  const int rb = (int)((rows + kFp8Block - 1) / kFp8Block), kb = (K + kFp8Block - 1) / kFp8Block;
  const int64_t total = count * rb * kb;
  const int64_t most = (int64_t)sms * 8;   // up to four CTAs of 512 threads an SM, two rounds
  quantize_fp8_blocks_kernel<T><<<(unsigned)(total < most ? total : most), kBlockThreads, 0, stream>>>(
      static_cast<const T*>(x), rows, K, vec, power, q, scales, rb, kb, total);
}

template <typename T>
void launch_dequantize(const uint8_t* q, const float* scales, const Fp8ScaleStrides& st, int64_t count, int64_t rows,
                       int K, int shift, void* out, int sms, cudaStream_t stream) {
  const RowGrid g = row_grid(K / 16, count * rows, sms);
  dequantize_fp8_kernel<T><<<g.grid, g.block, 0, stream>>>(q, scales, st, rows, count * rows, K, shift,
                                                          static_cast<T*>(out));
}

bool fp8_dtype(int d) { return d == LMOE_DTYPE_BF16 || d == LMOE_DTYPE_F16 || d == LMOE_DTYPE_F32; }

}  // namespace
}  // namespace lmoe

using namespace lmoe;

extern "C" int lmoe_quantize_fp8(const void* x, int dtype, int64_t rows, int K, int64_t ldx, int power_of_two,
                                 const int32_t* positions, int copies, int64_t out_rows, uint8_t* q, float* scales,
                                 int64_t scale_pitch, lmoe_stream_t stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  LMOE_ARG_CHECK(fp8_dtype(dtype));
  LMOE_ARG_CHECK(rows >= 0 && K > 0 && K % 16 == 0 && K <= kMaxColumns && ldx >= K && out_rows >= 0 && scale_pitch >= out_rows);
  LMOE_ARG_CHECK(positions ? copies >= 1 : (copies == 1 && out_rows == rows));
  if (rows == 0) return LMOE_OK;
  LMOE_ARG_CHECK(x && q && scales && aligned16(q) && (reinterpret_cast<uintptr_t>(scales) & 3) == 0);
  LMOE_ARG_CHECK((reinterpret_cast<uintptr_t>(positions) & 3) == 0);
  const int64_t esize = dtype == LMOE_DTYPE_F32 ? 4 : 2;
  LMOE_ARG_CHECK(reinterpret_cast<uintptr_t>(x) % esize == 0);
  Fp8RowArgs a;
  a.x = x;
  a.ldx = ldx;
  a.rows = rows;
  a.K = K;
  a.power_of_two = power_of_two;
  a.positions = positions;
  a.copies = copies;
  a.out_rows = out_rows;
  a.q = q;
  a.scales = scales;
  a.pitch = scale_pitch;
  a.vec = vector_bytes(x, ldx * esize);
  DeviceInfo dev;
  const int st = get_device_info(&dev);
  if (st != LMOE_OK) return st;
  const int wide = dtype == LMOE_DTYPE_F32 ? 16 : 32;   // columns of a thread
  const RowGrid g = row_grid((K + wide - 1) / wide, rows, dev.num_sms);
  if (dtype == LMOE_DTYPE_BF16)
    quantize_fp8_rows_kernel<__nv_bfloat16><<<g.grid, g.block, 0, stream>>>(a);
  else if (dtype == LMOE_DTYPE_F16)
    quantize_fp8_rows_kernel<__half><<<g.grid, g.block, 0, stream>>>(a);
  else
    quantize_fp8_rows_kernel<float><<<g.grid, g.block, 0, stream>>>(a);
  return cuda_status(cudaGetLastError());
}

extern "C" int lmoe_quantize_fp8_blocks(const void* x, int dtype, int64_t count, int64_t rows, int K, int power_of_two,
                                        uint8_t* q, float* scales, lmoe_stream_t stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  LMOE_ARG_CHECK(fp8_dtype(dtype));
  LMOE_ARG_CHECK(count >= 0 && rows >= 0 && rows <= INT32_MAX - kFp8Block && K > 0 && K % 16 == 0 && K <= kMaxColumns);
  if (count == 0 || rows == 0) return LMOE_OK;
  LMOE_ARG_CHECK(x && q && scales && aligned16(q) && (reinterpret_cast<uintptr_t>(scales) & 3) == 0);
  const int64_t esize = dtype == LMOE_DTYPE_F32 ? 4 : 2;
  LMOE_ARG_CHECK(reinterpret_cast<uintptr_t>(x) % esize == 0);
  DeviceInfo dev;
  const int st = get_device_info(&dev);
  if (st != LMOE_OK) return st;
  const int vec = vector_bytes(x, (int64_t)K * esize);
  if (dtype == LMOE_DTYPE_BF16)
    launch_blocks<__nv_bfloat16>(x, rows, K, vec, power_of_two, q, scales, count, dev.num_sms, stream);
  else if (dtype == LMOE_DTYPE_F16)
    launch_blocks<__half>(x, rows, K, vec, power_of_two, q, scales, count, dev.num_sms, stream);
  else
    launch_blocks<float>(x, rows, K, vec, power_of_two, q, scales, count, dev.num_sms, stream);
  return cuda_status(cudaGetLastError());
}

extern "C" int lmoe_dequantize_fp8(const uint8_t* q, const float* scales, int64_t scale_mat_stride,
                                   int64_t scale_row_stride, int64_t scale_block_stride, int64_t count, int64_t rows,
                                   int K, int block_rows, int out_dtype, void* out, lmoe_stream_t stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  LMOE_ARG_CHECK(fp8_dtype(out_dtype));
  LMOE_ARG_CHECK(block_rows == 1 || block_rows == kFp8Block);
  LMOE_ARG_CHECK(count >= 0 && rows >= 0 && K > 0 && K % 16 == 0 && K <= kMaxColumns);
  LMOE_ARG_CHECK(scale_mat_stride >= 0 && scale_row_stride >= 0 && scale_block_stride >= 0);
  if (count == 0 || rows == 0) return LMOE_OK;
  LMOE_ARG_CHECK(q && scales && out && aligned16(out) && aligned16(q) &&
                 (reinterpret_cast<uintptr_t>(scales) & 3) == 0);
  DeviceInfo dev;
  const int status = get_device_info(&dev);
  if (status != LMOE_OK) return status;
  const Fp8ScaleStrides st = {scale_mat_stride, scale_row_stride, scale_block_stride};
  const int shift = block_rows == 1 ? 0 : 7;
  if (out_dtype == LMOE_DTYPE_BF16)
    launch_dequantize<__nv_bfloat16>(q, scales, st, count, rows, K, shift, out, dev.num_sms, stream);
  else if (out_dtype == LMOE_DTYPE_F16)
    launch_dequantize<__half>(q, scales, st, count, rows, K, shift, out, dev.num_sms, stream);
  else
    launch_dequantize<float>(q, scales, st, count, rows, K, shift, out, dev.num_sms, stream);
  return cuda_status(cudaGetLastError());
}
