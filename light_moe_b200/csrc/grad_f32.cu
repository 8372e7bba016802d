// grad_f32.cu -- the gradients of the grouped product, and the product of any row length, for fp32
// operands of few rows per expert, on CUDA cores.
//
//   input gradient   dx[r, k]    = sum_n dy[r, n] * w[e(r), n, k]
//   weight gradient  dw[e, n, k] = sum_{r in e} dy[r, n] * x[r, k]
//   product          y[r, n]     = sum_k x[r, k] * w[e(r), n, k]
//
// With few rows, writing the operands as bf16 planes for the tensor cores (grad_split.cu) costs
// more than the products.  As in simt_gemm.cu, fp32 operands are multiplied and summed with fp32
// FFMA in contraction order.  Bound by the FFMA
// rate.  Tiles of 128 x 128 outputs, 16 contraction values per step in shared memory (the next
// step's loads are in registers meanwhile), 256 threads of 8 x 8 outputs: 16 shared-memory words
// feed 64 FFMAs.  Any size: operands whose rows are not multiples of 16 bytes are read word by
// word.
#include "grad_gemm.h"
#include "host_util.h"
#include "pair_gemm.cuh"

namespace lmoe {
namespace {

constexpr int kT = 128, kTK = 16, kNT = 256;
constexpr uint32_t kSite = 0xa00u;

struct F32Args {
  const float* dy;      // [R, N]
  const float* other;   // w [E, N, K] or x [R, K]
  const void* offsets;
  int offsets_i64;
  int E, N, K;
  int64_t R;
  int MT;
  Raster raster;
  float* out;
  uint32_t* err;
};

// Four consecutive values of a row from column c (zero from column `cols` on).
template <bool VEC>
__device__ __forceinline__ float4 load4(const float* row, int c, int cols) {
  if (VEC) return c < cols ? __ldg(reinterpret_cast<const float4*>(row + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
  float4 v;
  v.x = c < cols ? __ldg(row + c) : 0.f;
  v.y = c + 1 < cols ? __ldg(row + c + 1) : 0.f;
  v.z = c + 2 < cols ? __ldg(row + c + 2) : 0.f;
  v.w = c + 3 < cols ? __ldg(row + c + 3) : 0.f;
  return v;
}

template <int FORM, bool VEC>
__global__ void __launch_bounds__(kNT, 2) grad_f32_kernel(const F32Args a) {
  constexpr bool WGRAD = FORM == kGradWeight, kProduct = FORM == kGradProduct;
  __shared__ SegTable seg;
  __shared__ __align__(16) float as[kTK][kT + 4];
  __shared__ __align__(16) float bs[kTK][kT + 4];
  const int tid = threadIdx.x;
  load_segments(&seg, a.offsets, a.offsets_i64, a.E, a.R, tid, kNT);
  const int segs = a.E + 2;
  if (tid < 32)
    scan_tiles(&seg, segs, tid, [&](int j) {
      if (!WGRAD) return (seg.row[j + 1] - seg.row[j] + kT - 1) / kT * a.raster.nb;
      return j == 0 || j == a.E + 1 ? 0 : a.MT * a.raster.nb;
    });
  if (tid == 0 && seg.bad && blockIdx.x == 0) report_error(a.err, kErrBadArg, kSite + 1);
  __syncthreads();
  const int total = seg.tile_start[segs];
  const int tx = tid & 15, ty = tid >> 4;
  int j = 0;
  for (int tile = blockIdx.x; tile < total; tile += gridDim.x) {
    while (tile >= seg.tile_start[j + 1]) ++j;
    const int rows = seg.row[j + 1] - seg.row[j];
    int m, n;
    a.raster.at(tile - seg.tile_start[j], WGRAD ? a.MT : (rows + kT - 1) / kT, m, n);
    const int e = j - 1;
    const bool zero = j == 0 || j == a.E + 1;
    const int r0 = seg.row[j] + (WGRAD ? 0 : m * kT);
    const int m_rows = WGRAD ? min(kT, a.N - m * kT) : min(kT, seg.row[j + 1] - r0);
    const int depth = zero ? 0 : (WGRAD ? rows : a.N);
    const int c0 = n * kT;
    // contraction row d of B: w[e, d, :] or x[r0 + d, :]; the product: row c of w[e], d along it
    const float* bbase = a.other + (WGRAD ? (int64_t)r0 * a.K : (int64_t)(zero ? 0 : e) * a.N * a.K);
    const float* abase = a.dy + (int64_t)r0 * a.N;
    float4 av[2], bv[2];
    auto load = [&](int d0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int idx = tid + i * kNT;
        const int d = d0 + (idx >> 5), c = (idx & 31) * 4;   // 32 quads of columns a contraction row
        const int r = idx >> 2, q = (idx & 3) * 4;           // four quads of contraction values a row
        if (kProduct)
          bv[i] = c0 + r < a.K ? load4<VEC>(bbase + (int64_t)(c0 + r) * a.N, d0 + q, depth)
                               : make_float4(0.f, 0.f, 0.f, 0.f);
        else
          bv[i] = d < depth ? load4<VEC>(bbase + (int64_t)d * a.K, c0 + c, a.K) : make_float4(0.f, 0.f, 0.f, 0.f);
        if (WGRAD) {
          av[i] = d < depth ? load4<VEC>(abase + (int64_t)d * a.N, m * kT + c, a.N) : make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
          av[i] = r < m_rows ? load4<VEC>(abase + (int64_t)r * a.N, d0 + q, depth) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
    };
    float acc[8][8];
#pragma unroll
    for (int y = 0; y < 8; ++y)
#pragma unroll
      for (int x = 0; x < 8; ++x) acc[y][x] = 0.0f;
    if (depth > 0) load(0);
    for (int d0 = 0; d0 < depth; d0 += kTK) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int idx = tid + i * kNT;
        const int r = idx >> 2, q = (idx & 3) * 4;
        if (kProduct) {
          bs[q][r] = bv[i].x;
          bs[q + 1][r] = bv[i].y;
          bs[q + 2][r] = bv[i].z;
          bs[q + 3][r] = bv[i].w;
        } else {
          *reinterpret_cast<float4*>(&bs[idx >> 5][(idx & 31) * 4]) = bv[i];
        }
        if (WGRAD) {
          *reinterpret_cast<float4*>(&as[idx >> 5][(idx & 31) * 4]) = av[i];
        } else {
          as[q][r] = av[i].x;
          as[q + 1][r] = av[i].y;
          as[q + 2][r] = av[i].z;
          as[q + 3][r] = av[i].w;
        }
      }
      __syncthreads();
      if (d0 + kTK < depth) load(d0 + kTK);
#pragma unroll
      for (int kk = 0; kk < kTK; ++kk) {
        float ra[8], rb[8];
        *reinterpret_cast<float4*>(ra) = *reinterpret_cast<const float4*>(&as[kk][ty * 4]);
        *reinterpret_cast<float4*>(ra + 4) = *reinterpret_cast<const float4*>(&as[kk][64 + ty * 4]);
        *reinterpret_cast<float4*>(rb) = *reinterpret_cast<const float4*>(&bs[kk][tx * 4]);
        *reinterpret_cast<float4*>(rb + 4) = *reinterpret_cast<const float4*>(&bs[kk][64 + tx * 4]);
#pragma unroll
        for (int y = 0; y < 8; ++y)
#pragma unroll
          for (int x = 0; x < 8; ++x) acc[y][x] = __fmaf_rn(ra[y], rb[x], acc[y][x]);
      }
      __syncthreads();
    }
#pragma unroll
    for (int y = 0; y < 8; ++y) {
      const int r = (y & 4) * 16 + ty * 4 + (y & 3);
      if (r >= m_rows) continue;
      float* row = a.out + (WGRAD ? (int64_t)e * a.N + m * kT + r : (int64_t)r0 + r) * a.K;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = c0 + h * 64 + tx * 4;
        if (VEC) {
          if (c < a.K)
            *reinterpret_cast<float4*>(row + c) =
                make_float4(acc[y][4 * h], acc[y][4 * h + 1], acc[y][4 * h + 2], acc[y][4 * h + 3]);
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (c + x < a.K) row[c + x] = acc[y][4 * h + x];
        }
      }
    }
  }
}

}  // namespace

int run_grad_f32(const GradProblem& p, cudaStream_t stream) {
  DeviceInfo dev;
  const int st = get_device_info(&dev);
  if (st != LMOE_OK) return st;
  F32Args a = {};
  a.dy = static_cast<const float*>(p.dy);
  a.other = static_cast<const float*>(p.other);
  a.offsets = p.offsets;
  a.offsets_i64 = p.offsets_i64;
  a.E = p.num_experts;
  a.N = p.N;
  a.K = p.K;
  a.R = p.total_rows;
  a.MT = (p.N + kT - 1) / kT;
  a.raster = Raster((p.K + kT - 1) / kT);
  a.out = static_cast<float*>(p.out);
  a.err = p.err;
  const bool vec = p.N % 4 == 0 && p.K % 4 == 0 && aligned16(p.dy) && aligned16(p.other) && aligned16(p.out);
  const int grid = dev.num_sms * 2;   // two CTAs fit an SM's registers
  auto fn = p.form == kGradWeight    ? (vec ? grad_f32_kernel<kGradWeight, true> : grad_f32_kernel<kGradWeight, false>)
            : p.form == kGradInput   ? (vec ? grad_f32_kernel<kGradInput, true> : grad_f32_kernel<kGradInput, false>)
                                     : (vec ? grad_f32_kernel<kGradProduct, true> : grad_f32_kernel<kGradProduct, false>);
  fn<<<grid, kNT, 0, stream>>>(a);
  return cuda_status(cudaGetLastError());
}

}  // namespace lmoe
