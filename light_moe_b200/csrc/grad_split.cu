// grad_split.cu -- the gradients of grad_gemm.cu (and the product of any row length) for fp32 operands
// on tensor cores (sm_100a).
//
// A value is the sum of three bf16 planes, x = high + middle + low to 2^-26 (but not below 2^-134, half
// of the smallest bf16), and a product of two
// values the sum of the six products of planes down to 2^-18: (m, m), (l, h), (h, l), (m, h),
// (h, m), (h, h); six times the bf16 work at ~16 times the FFMA rate.  The tensor pipe truncates
// its sums (measured: 1024 bf16 products of mean 1 come out 8e-7 low, 8192 2.5e-5), so a TMEM
// accumulator takes 64 contraction values only, small products first, and the epilogue adds the
// accumulators in registers, rounding to nearest.
//
// A stage holds 64 contraction values of all planes of both operands (16 KB a plane of 128 rows or
// columns), so that each is loaded once for its products; two or three stages, two accumulators.  (With a
// stage for each pair of planes the copies bound it: dx of 1021 rows on 8 experts of 1024 x 2816
// 120 us.)
//
// Activations (dy, x) are written as planes by a pass of their own: a row is read by every column
// tile.  Weights are not: in the input gradient and the product eight warps read a tile's fp32
// values two stages ahead into registers and write their planes into shared memory, which saves
// writing and reading 12 bytes a weight.  Their tiles are 256 x 128, so that planes and registers
// fit; the weight gradient's are 256 x 256 or, where the last round would leave pairs idle, 256 x
// 128.  The weights' values are split before their stage is free, so that only eight-byte stores lie
// between one stage's MMAs and the next (four warps that split them afterwards, two stages: 108
// against 83 us for dx of 1021 rows on 8 experts of 1024 x 2816).
//
// For those sizes the weight gradient takes 52 us: 14 for writing 92 MB, ~16 for the MMAs, the planes'
// pass and the launches.  The input gradient is bound by shared memory (an MMA of 128 columns reads
// operands in all of its 64 cycles, the copies and planes come on top) and, with few rows per expert,
// by the tile's empty rows.
//
// Warps: 0 TMA producer; 1 MMA issuer (leader CTA); 2 clears the tails of segments (weight
// gradient); 4-11 epilogue, eight warps of 32 rows x half the columns; 12-19 weights.
#include <cuda_bf16.h>

#include "grad_tile.cuh"

namespace lmoe {
namespace {

constexpr int kSK = 64;            // contraction values per stage
constexpr int kAcc = 2;
constexpr int kEpiWarp0 = 4, kEpiWarps = 8, kConvWarp0 = 12, kConvWarps = 8;
constexpr uint32_t kChunk = 64 * 128;             // 64 lines of 64 values
constexpr uint32_t kPlane = 2 * kChunk;           // a plane of 128 rows or columns
constexpr uint32_t kSite = 0x700u;
// The products of planes (0 high, 1 middle, 2 low), in their order.
constexpr int kPairs = 6;
constexpr uint32_t kPlaneA = 0x001021, kPlaneB = 0x010201;   // hex digit i: of product i

template <int FORM>
struct Cfg {
  static constexpr bool kConv = FORM != kGradWeight;   // weights converted in the kernel
  static constexpr int kThreads = (kConv ? kConvWarp0 + kConvWarps : kConvWarp0) * 32;
  static constexpr uint32_t kPlaneOfB = kConv ? kChunk : kPlane;
  static constexpr uint32_t kStageBytes = 3 * (kPlane + kPlaneOfB);
  static constexpr int kStages = kConv ? 3 : 2;
  // a warp's block on its way out (weights converted: rows of odd lengths only)
  static constexpr uint32_t kBlockBytes = kConv ? 32 * 32 : 32 * 128;
  static constexpr int kBlocks = kConv ? 2 : 4;        // blocks of 32 columns of an epilogue warp
};

template <int kStages>
struct __align__(8) Bars {
  uint64_t full[kStages];       // leader: both CTAs' operands landed (and weights were converted)
  uint64_t empty[kStages];      // the stage's MMAs finished (both CTAs)
  uint64_t tail[kStages];       // this CTA's operands of a stage with a tail to clear
  uint64_t acc_full[kAcc];
  uint64_t acc_empty[kAcc];     // leader: both CTAs' epilogue warps
  uint64_t mma_done;
  uint32_t tmem_base;
  int abort;
  SegTable seg;
};

// Whether a stage with `left` rows of its segment ends inside the 16 rows of an MMA.
__device__ __forceinline__ bool has_tail(int left) { return left < kSK && (left & 15) != 0; }

// The planes of two values.  Rounding each remainder to nearest leaves at most 2^-27 of the value.
__device__ __forceinline__ void split2(float x, float y, uint32_t (&w)[3]) {
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    w[k] = *reinterpret_cast<const uint32_t*>(&h);
    x = __fsub_rn(x, __uint_as_float(w[k] << 16));   // exact
    y = __fsub_rn(y, __uint_as_float(w[k] & 0xffff0000u));
  }
}
// Four values.  Values that would round to an infinity are cut instead; values that are not finite
// stay in the high plane.
__device__ __forceinline__ void split4(const float4 v, uint32_t (&lo)[3], uint32_t (&hi)[3]) {
  const float f[4] = {v.x, v.y, v.z, v.w};
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = __float_as_uint(f[i]) & 0x7fffffffu;
    top = b > top ? b : top;
  }
  if (top < 0x7f7f8000u) {   // all round to finite values
    split2(f[0], f[1], lo);
    split2(f[2], f[3], hi);
    return;
  }
  uint32_t b[4][3];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool finite = (__float_as_uint(f[i]) & 0x7f800000u) != 0x7f800000u;
    const __nv_bfloat16 h = finite ? __float2bfloat16_rz(f[i]) : __float2bfloat16_rn(f[i]);
    const float e = finite ? __fsub_rn(f[i], __bfloat162float(h)) : 0.0f;
    const __nv_bfloat16 m = __float2bfloat16_rn(e);
    b[i][0] = __bfloat16_as_ushort(h);
    b[i][1] = __bfloat16_as_ushort(m);
    b[i][2] = __bfloat16_as_ushort(__float2bfloat16_rn(__fsub_rn(e, __bfloat162float(m))));
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    lo[k] = b[0][k] | b[1][k] << 16;
    hi[k] = b[2][k] | b[3][k] << 16;
  }
}

// Four values from row r, column c of a matrix; zeros outside.
__device__ __forceinline__ float4 load4(const float* src, int64_t ld, int r, int c, int rows, int cols, bool vec) {
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (r >= rows || c >= cols) return v;
  const float* p = src + r * ld + c;
  if (vec) return __ldg(reinterpret_cast<const float4*>(p));   // whole: the row length is a multiple of 4
  v.x = __ldg(p);
  if (c + 1 < cols) v.y = __ldg(p + 1);
  if (c + 2 < cols) v.z = __ldg(p + 2);
  if (c + 3 < cols) v.w = __ldg(p + 3);
  return v;
}

template <int FORM>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Cfg<FORM>::kThreads, 1)
    grad_split_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_a32,
                      const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_out,
                      const float* weights, int vec, const GradArgs a) {
  using C = Cfg<FORM>;
  using B = Bars<C::kStages>;
  constexpr int kStages = C::kStages;
  constexpr uint32_t kBlockBytes = C::kBlockBytes;
  extern __shared__ __align__(1024) uint8_t base[];   // whole swizzle atoms
  uint8_t* store_stage = base + kStages * C::kStageBytes;
  B* bars = reinterpret_cast<B*>(store_stage + kEpiWarps * kBlockBytes);
  volatile int* abort_flag = &bars->abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars->full[s], C::kConv ? 2 + 2 * kConvWarps : 2);
      mbar_init(&bars->empty[s], 1);
      mbar_init(&bars->tail[s], 1);
    }
    for (int s = 0; s < kAcc; ++s) {
      mbar_init(&bars->acc_full[s], 1);
      mbar_init(&bars->acc_empty[s], 2 * kEpiWarps);
    }
    mbar_init(&bars->mma_done, 1);
    bars->abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(&bars->tmem_base, 512);
    tmem_relinquish_pair();
  }
  load_segments(&bars->seg, a.offsets, a.offsets_i64, a.E, a.R, tid, C::kThreads);
  const int segs = a.E + 2;
  if (warp == 0)
    scan_tiles(&bars->seg, segs, lane, [&](int j) {
      if (FORM != kGradWeight) return (bars->seg.row[j + 1] - bars->seg.row[j] + kTile - 1) / kTile * a.raster.nb;
      return j == 0 || j == a.E + 1 ? 0 : a.MT * a.raster.nb;
    });
  if (tid == 0 && bars->seg.bad && blockIdx.x == 0) report_error(a.err, kErrBadArg, kSite + 1);
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  const SegTable& seg = bars->seg;
  const int total = seg.tile_start[segs];
  const int first = blockIdx.x >> 1, stride = gridDim.x >> 1;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    const uint32_t full_addr = mapa_u32(&bars->full[0], 0);
    Ring<kStages> st;
    int hint = 0;
    bool ok = true;
    for (int tile = first; tile < total && ok; tile += stride) {
      const Tile t = tile_at<FORM, kSK>(seg, a, tile, hint);
      const int c0 = t.n * a.width + (int)rank * (a.width / 2);   // first column of B
      const int m0 = (FORM != kGradWeight ? t.row0 : t.m * kTile) + (int)rank * kCta;
      const int rows = t.row_end - m0;
      // 32-row boxes of dy that hold this CTA's rows (not the weight gradient)
      const int boxes = rows <= 0 ? 0 : (rows >= kCta ? 4 : (rows + 31) >> 5);
      const bool wide = a.width == kTile;
      for (int ks = 0; ks < t.ks; ++ks, st.next()) {
        ok = warp_wait(&bars->empty[st.i], st.phase ^ 1u, a.err, abort_flag, kSite + 2);
        if (!ok) break;
        if (elect_one()) {
          uint8_t* sa = base + st.i * C::kStageBytes;
          const uint32_t bar = full_addr + st.i * 8;
          if constexpr (FORM != kGradWeight) {
            mbar_arrive_expect_tx_cluster(bar, (uint32_t)boxes * 3u * 4096u);
            for (int p = 0; p < 3; ++p) {
              const int y = m0 + p * (int)a.R;
              if (boxes == 4) {
                tma_load_2d_pair(sa + p * kPlane, &tm_a, bar, ks * kSK, y);
              } else {
                for (int b = 0; b < boxes; ++b)
                  tma_load_2d_pair(sa + p * kPlane + b * 4096, &tm_a32, bar, ks * kSK, y + b * 32);
              }
            }
          } else {
            uint8_t* sb = sa + 3 * kPlane;
            const int r = t.row0 + ks * kSK;
            const uint32_t bytes = 3u * (kPlane + (wide ? kPlane : kChunk));
            if (has_tail(t.row_end - r)) {
              uint64_t* own = &bars->tail[st.i];
              mbar_arrive_expect_tx(own, bytes);
              for (int p = 0; p < 3; ++p) {
                const int y = r + p * (int)a.R;
                tma_load_2d(sa + p * kPlane, &tm_a, own, m0, y);
                tma_load_2d(sa + p * kPlane + kChunk, &tm_a, own, m0 + 64, y);
                tma_load_2d(sb + p * kPlane, &tm_b, own, c0, y);
                if (wide) tma_load_2d(sb + p * kPlane + kChunk, &tm_b, own, c0 + 64, y);
              }
            } else {
              mbar_arrive_expect_tx_cluster(bar, bytes);
              for (int p = 0; p < 3; ++p) {
                const int y = r + p * (int)a.R;
                tma_load_2d_pair(sa + p * kPlane, &tm_a, bar, m0, y);
                tma_load_2d_pair(sa + p * kPlane + kChunk, &tm_a, bar, m0 + 64, y);
                tma_load_2d_pair(sb + p * kPlane, &tm_b, bar, c0, y);
                if (wide) tma_load_2d_pair(sb + p * kPlane + kChunk, &tm_b, bar, c0 + 64, y);
              }
            }
          }
        }
      }
    }
    // the copies of a finished tile have landed (its MMAs read them)
    if (!ok) let_copies_land();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (leader) {
      const uint32_t idesc = idesc_f16kind_f32(kTile, a.width, 0) | (FORM == kGradProduct ? 0u : kIdescBMajorMN) |
                             (FORM == kGradWeight ? kIdescAMajorMN : 0u);
      // descriptors count 16 bytes
      const uint32_t sa = smem_u32(base), sb = sa + 3 * kPlane;
      const uint64_t adesc0 = FORM != kGradWeight ? sdesc_k_sw128(sa) : sdesc_mn_sw128(sa, kChunk);
      const uint64_t bdesc0 = FORM == kGradProduct ? sdesc_k_sw128(sb) : sdesc_mn_sw128(sb, kChunk);
      Ring<kStages> st;
      Ring<kAcc> ac;
      int hint = 0;
      bool ok = true;
      for (int tile = first; tile < total && ok; tile += stride) {
        const Tile t = tile_at<FORM, kSK>(seg, a, tile, hint);
        const int depth = FORM != kGradWeight ? a.N : t.row_end - t.row0;
        for (int ks = 0; ks < t.ks; ++ks, st.next(), ac.next()) {
          ok = warp_wait(&bars->acc_empty[ac.i], ac.phase ^ 1u, a.err, abort_flag, kSite + 4) &&
               warp_wait(&bars->full[st.i], st.phase, a.err, abort_flag, kSite + 6);
          if (!ok) break;
          tc_fence_after();
          const int left = depth - ks * kSK;
          if (elect_one()) {
            const uint32_t d = tmem + ac.i * kTile;
            const uint64_t ad = adesc0 + st.i * (C::kStageBytes >> 4), bd = bdesc0 + st.i * (C::kStageBytes >> 4);
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
              const uint32_t pa = (kPlaneA >> (4 * i) & 15u) * (kPlane >> 4);
              const uint32_t pb = (kPlaneB >> (4 * i) & 15u) * (C::kPlaneOfB >> 4);
#pragma unroll
              for (int kk = 0; kk < kSK / 16; ++kk) {
                // 16 contraction values: 32 bytes of the lines of a K-major plane, or 16 lines
                const uint32_t sta = FORM != kGradWeight ? kk * 2 : kk * 128;
                const uint32_t stb = FORM == kGradProduct ? kk * 2 : kk * 128;
                if (kk * 16 < left) mma_ss_pair(d, ad + pa + sta, bd + pb + stb, idesc, (i | kk) != 0 ? 1u : 0u);
              }
            }
            mma_commit_pair(&bars->empty[st.i]);
            mma_commit_pair(&bars->acc_full[ac.i]);
          }
          __syncwarp();
        }
      }
      if (elect_one()) mma_commit_leader(&bars->mma_done);
      mbar_wait(&bars->mma_done, 0, a.err, nullptr, kSite + 7);
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ segment tails
    if (FORM == kGradWeight) {
      Ring<kStages> st;
      uint32_t tail_parity = 0;   // a bit per stage
      int hint = 0;
      bool ok = true;
      for (int tile = first; tile < total && ok; tile += stride) {
        const Tile t = tile_at<FORM, kSK>(seg, a, tile, hint);
        const int left = t.row_end - t.row0 - (t.ks - 1) * kSK;   // rows of the last stage
        for (int ks = 0; ks < t.ks; ++ks, st.next()) {
          if (ks != t.ks - 1 || !has_tail(left)) continue;
          ok = warp_wait(&bars->tail[st.i], tail_parity >> st.i & 1u, a.err, abort_flag, kSite + 8);
          if (!ok) break;
          tail_parity ^= 1u << st.i;
          // contraction rows [left, next multiple of 16) of the stage's chunks; a row is one
          // 128-byte line, which the swizzle only permutes
          const int m = (16 - (left & 15)) * 8;
          uint8_t* at = base + st.i * C::kStageBytes + left * 128;
          for (int c = 0; c < (int)(C::kStageBytes / kChunk); ++c)
            for (int k = lane; k < m; k += 32)
              *reinterpret_cast<uint4*>(at + c * kChunk + k * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_u32(&bars->full[st.i], 0));
        }
      }
    }
  } else if (warp >= kEpiWarp0 && warp < kConvWarp0) {
    // ------------------------------------------------------------------ epilogue
    const int q = warp & 3, half = (warp - kEpiWarp0) >> 2;
    const uint32_t lane_base = (uint32_t)(q * 32) << 16;
    const uint32_t empty_addr = mapa_u32(&bars->acc_empty[0], 0);
    const int64_t pitch = (int64_t)a.K * 4;
    uint8_t* stage = store_stage + (warp - kEpiWarp0) * kBlockBytes;
    Ring<kAcc> ac;
    int hint = 0;
    bool ok = true;
    for (int tile = first; tile < total; tile += stride) {
      const Tile t = tile_at<FORM, kSK>(seg, a, tile, hint);
      // the warp's 32 rows, and the first of its half of the columns
      const int r = (int)rank * kCta + q * 32;
      const int left = FORM != kGradWeight ? t.row_end - t.row0 - r : a.N - t.m * kTile - r;
      const int rows = left < 32 ? left : 32;
      const int64_t row = FORM != kGradWeight ? (int64_t)t.row0 + r : (int64_t)t.e * a.N + t.m * kTile + r;
      uint8_t* out = static_cast<uint8_t*>(a.out) + row * pitch;
      const int cols = a.width / 2;
      const int c0 = t.n * a.width + half * cols;
      const uint32_t col0 = tmem + lane_base + half * cols;
      // whole 32-row blocks leave by TMA; a weight gradient's rows behind N are cut by the tensor map
      const bool whole = !C::kConv && a.store != kStoreStaged && (FORM == kGradWeight ? rows > 0 : rows == 32);
      const int y = FORM == kGradWeight ? t.m * kTile + r : (int)row, z = FORM == kGradWeight ? t.e : 0;
      float f[C::kBlocks][32];
#pragma unroll
      for (int j = 0; j < C::kBlocks; ++j)
#pragma unroll
        for (int i = 0; i < 32; ++i) f[j][i] = 0.0f;
      for (int ks = 0; ks < t.ks; ++ks) {
        ok = warp_wait(&bars->acc_full[ac.i], ac.phase, a.err, abort_flag, kSite + 9);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int j = 0; j < 2 * C::kBlocks; ++j) {
          if (j * 16 >= cols) break;
          uint32_t u[16];
          tmem_ld16(col0 + ac.i * kTile + j * 16, u);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float& v = f[j >> 1][(j & 1) * 16 + i];
            v = __fadd_rn(v, __uint_as_float(u[i]));
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(empty_addr + ac.i * 8);
        ac.next();
      }
      if (!ok) break;
#pragma unroll
      for (int j = 0; j < C::kBlocks; ++j) {
        if (j * 32 >= cols || c0 + j * 32 >= a.K) break;
        if (!C::kConv && whole)
          store_block<128>(&tm_out, f[j], LMOE_DTYPE_F32, stage, lane, c0 + j * 32, y, z);
        else
          store_rows<32, kBlockBytes>(out, pitch, rows, c0 + j * 32, a.K, f[j], LMOE_DTYPE_F32, a.store, stage, lane);
      }
    }
    if (elect_one()) bulk_wait_all();   // the stores are complete
  } else if (C::kConv && warp >= kConvWarp0) {
    // ------------------------------------------------------------------ weights
    // A stage's 64 x 64 values, a warp two rows of 64 at a time: dx 64 contraction rows of 64
    // columns, the product 64 of its columns' rows of 64 contraction values.
    const int rows_of = FORM == kGradProduct ? a.K : a.N, cols_of = FORM == kGradProduct ? a.N : a.K;
    constexpr int kRows = 2 * kConvWarps, kPieces = 64 / kRows;   // rows at a time, values of four a lane
    const int r = (warp - kConvWarp0) * 2 + (lane >> 4), c = (lane & 15) * 4;
    const uint32_t full_addr = mapa_u32(&bars->full[0], 0);
    // its eight bytes of a line: 16-byte piece j of line r lies at j ^ (r & 7)
    uint8_t* dst = base + 3 * kPlane + r * 128 + (((lane & 15) >> 1) ^ (r & 7)) * 16 + (lane & 1) * 8;
    constexpr int kAhead = 2;
    float4 v[kAhead][kPieces];
    int pending = 0, hint = 0, ltile = first, lks = 0;   // the next load: tile and stage
    Tile lt = {};
    auto load = [&](float4 (&b)[kPieces]) {
      while (lks == 0) {   // the next tile that has an expert
        if (ltile >= total) return;
        lt = tile_at<FORM, kSK>(seg, a, ltile, hint);
        if (lt.ks != 0) break;
        ltile += stride;
      }
      const int across = lt.n * 128 + (int)rank * 64, along = lks * kSK;
      const int r0 = FORM == kGradProduct ? across : along, c0 = FORM == kGradProduct ? along : across;
      const float* src = weights + (int64_t)lt.e * rows_of * cols_of;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) b[i] = load4(src, cols_of, r0 + r + kRows * i, c0 + c, rows_of, cols_of, vec);
      ++pending;
      if (++lks == lt.ks) {
        lks = 0;
        ltile += stride;
      }
    };
#pragma unroll
    for (int j = 0; j < kAhead; ++j) load(v[j]);
    Ring<kStages> st;
    bool ok = true;
    while (ok && pending > 0) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (!ok || pending == 0) break;
        --pending;
        uint32_t lo[kPieces][3], hi[kPieces][3];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) split4(v[j][i], lo[i], hi[i]);
        load(v[j]);
        ok = warp_wait(&bars->empty[st.i], st.phase ^ 1u, a.err, abort_flag, kSite + 10);
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
#pragma unroll
          for (int p = 0; p < 3; ++p)
            *reinterpret_cast<uint2*>(dst + st.i * C::kStageBytes + p * C::kPlaneOfB + i * (kRows * 128)) =
                make_uint2(lo[i][p], hi[i][p]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(full_addr + st.i * 8);
        st.next();
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();   // the other CTA's arrivals and the MMAs on this CTA's memory are done
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

template <int FORM>
int launch(const CUtensorMap& ta, const CUtensorMap& ta32, const CUtensorMap& tb, const CUtensorMap& to,
           const float* weights, int vec, const GradArgs& a, int grid, cudaStream_t stream) {
  using C = Cfg<FORM>;
  constexpr size_t smem = C::kStages * C::kStageBytes + kEpiWarps * C::kBlockBytes + sizeof(Bars<C::kStages>);
  static_assert(smem <= 232448, "shared memory budget");
  static_assert(C::kStageBytes % 1024 == 0 && 2 * kConvWarps % 8 == 0, "swizzle atoms");
  auto fn = grad_split_kernel<FORM>;
  const int st = set_max_dynamic_smem(reinterpret_cast<const void*>(fn), smem);
  if (st != LMOE_OK) return st;
  fn<<<grid, C::kThreads, smem, stream>>>(ta, ta32, tb, to, weights, vec, a);
  return cuda_status(cudaGetLastError());
}

// The planes of src [rows, cols]: dst [3][rows, pitch] bf16, zero behind the columns.
__global__ void __launch_bounds__(256) split_rows_kernel(const __grid_constant__ CopyJobs jobs) {
  const CopyJob& job = jobs.job[blockIdx.y];
  const float* __restrict__ src = static_cast<const float*>(job.src);
  const int64_t rows = job.rows;
  const int cols = job.cols, pitch = job.pitch;
  const bool vec = cols % 4 == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0;
  uint4* __restrict__ dst = job.dst;
  const int per = pitch / 8;
  const int64_t total = rows * per;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / per;
    const int c = (int)(i - r * per) * 8;
    const float* row = src + r * cols;
    uint32_t w[4][3];
    split4(load4(row, 0, 0, c, 1, cols, vec), w[0], w[1]);
    split4(load4(row, 0, 0, c + 4, 1, cols, vec), w[2], w[3]);
#pragma unroll
    for (int k = 0; k < 3; ++k) dst[k * total + i] = make_uint4(w[0][k], w[1][k], w[2][k], w[3][k]);
  }
}

}  // namespace

bool grad_splits(const GradProblem& p) {
  // Beside the planes' passes and the launches (~10 us) the tensor cores win.  us on CUDA cores against
  // planes, E x N x K: input gradient, 4 rows an expert, 8 x 32 x 256 8.4 : 12.5, 8 x 96 x 256 14.6 :
  // 14.5, 8 x 128 x 128 18.7 : 14.5, 8 x 1024 x 2816 199 : 70 (its tiles there cost what full ones do);
  // 64 rows, 8 x 64 x 2816 17.4 : 20.7.  Weight gradient, 64 x 128 x 512, 64 rows 22.9 : 26.9; 4 x 2048 x
  // 2048, 1 row 27 : 33, 16 rows 29 : 28, 24 rows 41 : 29; 64 x 512 x 1024, 1 row 50 : 39.
  if (p.dtype != LMOE_DTYPE_F32 || p.total_rows * 3 > INT32_MAX) return false;
  const double weights = (double)p.N * p.K, work = (double)p.total_rows * weights;
  if (work > 1 << 28) return true;
  return weight_grad(p) ? weights * p.num_experts > 1 << 24 : p.N >= 96;
}

size_t grad_split_workspace(const GradProblem& p) {
  if (!grad_splits(p)) return 0;
  return align256((size_t)p.total_rows * pitch8(p.N) * 6) +
         (weight_grad(p) ? align256((size_t)p.total_rows * pitch8(p.K) * 6) : 0);
}

int run_grad_split(const GradProblem& p, cudaStream_t stream) {
  DeviceInfo dev;
  int st = get_device_info(&dev);
  if (st != LMOE_OK) return st;
  if (dev.cc_major != 10) return LMOE_ERR_DEVICE;
  const int64_t ldy = pitch8(p.N), ldx = pitch8(p.K);
  uint8_t* dy = static_cast<uint8_t*>(p.workspace);
  uint8_t* x = dy + align256((size_t)p.total_rows * ldy * 6);
  CopyJobs jobs = {};
  jobs.add(p.dy, p.total_rows, p.N, ldy, dy);
  if (weight_grad(p)) jobs.add(p.other, p.total_rows, p.K, ldx, x);
  split_rows_kernel<<<jobs.grid(dev), 256, 0, stream>>>(jobs);
  st = cuda_status(cudaGetLastError());
  if (st != LMOE_OK) return st;
  GradArgs a = {};
  CUtensorMap ta, ta32, tb, to = {};
  st = fill_args(p, kSK, 1, a, to);
  if (st != LMOE_OK) return st;
  const int grid = gemm_grid(dev) < 2 ? 2 : gemm_grid(dev) & ~1;   // whole pairs
  const CUtensorMapDataType dt = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint64_t rows = 3 * (uint64_t)p.total_rows;   // of the planes, one behind the other
  // the maps end at the true sizes, so that TMA fills what lies behind them with zeros
  if (weight_grad(p)) {
    const int widths[] = {256, 128};
    a.width = pick_width(widths, grid / 2, 0, 16,
                         [&](int w) { return (int64_t)a.MT * p.num_experts * ((p.K + w - 1) / w); });
    a.raster = Raster((p.K + a.width - 1) / a.width);
    st = encode_tmap_2d(&ta, dy, dt, 2, rows, (uint64_t)p.N, (uint64_t)ldy * 2, 64, 64, true);
    if (st != LMOE_OK) return st;
    st = encode_tmap_2d(&tb, x, dt, 2, rows, (uint64_t)p.K, (uint64_t)ldx * 2, 64, 64, true);
    if (st != LMOE_OK) return st;
    return launch<kGradWeight>(ta, ta, tb, to, nullptr, 0, a, grid, stream);
  }
  a.width = 128;
  a.raster = Raster((p.K + a.width - 1) / a.width);
  st = encode_tmap_2d(&ta, dy, dt, 2, rows, (uint64_t)p.N, (uint64_t)ldy * 2, kCta, 64, true);
  if (st != LMOE_OK) return st;
  st = encode_tmap_2d(&ta32, dy, dt, 2, rows, (uint64_t)p.N, (uint64_t)ldy * 2, 32, 64, true);
  if (st != LMOE_OK) return st;
  const float* w = static_cast<const float*>(p.other);
  const int vec = other_cols(p) % 4 == 0 && aligned16(w);
  return p.form == kGradProduct ? launch<kGradProduct>(ta, ta32, ta, to, w, vec, a, grid, stream)
                                : launch<kGradInput>(ta, ta32, ta, to, w, vec, a, grid, stream);
}

}  // namespace lmoe
