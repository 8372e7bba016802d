// grad_gemm.cu -- the two gradients of the grouped product y[r, n] = sum_k x[r, k] * w[e, n, k]
// over ragged row segments, and the product itself for any row length, on CTA pairs (sm_100a).
//
//   input gradient   dx[r, k]    = sum_n dy[r, n] * w[e(r), n, k]        contraction over n
//   weight gradient  dw[e, n, k] = sum_{r in e} dy[r, n] * x[r, k]       contraction over rows
//   product          y[r, n]     = sum_k x[r, k] * w[e(r), n, k]         contraction over k
//                    (grouped_gemm.cu has it for k a multiple of 128)
//
// None needs a transposed copy: an operand whose contraction index is the slow one in memory
// (w and both operands of dw) is loaded by TMA as it lies, in chunks of 64 columns x 128
// contraction rows, and read by tcgen05.mma as an M- or N-major operand.
//
// Tile: 256 x 256 on a CTA pair (128 rows of A and 128 columns of B per CTA), two accumulators
// of 256 columns fill the 512 TMEM columns, three stages of 128 contraction values (64 KB per CTA:
// a stage costs the issuing warp ~600 cycles beside its MMAs, so they are few and long); 256 x 128
// where the last round of tiles would leave pairs idle.
// Bound by the tensor pipe for prompt-sized segments (8192 rows, 8 experts of 14336 x 4096: dx 713, dw 703
// us, 1.36 PFLOP/s); with few rows per expert the input gradient is bound by reading w and the weight
// gradient by writing dw (HBM; 12288 rows on 64 experts of 1408 x 2048, uneven: 95 and 106 us).
//
// A segment's rows need not end at a stage: the rows of the next expert (or beyond) in the last
// stage of a weight gradient are cleared in shared memory, in both operands, before its MMAs --
// a product with a zero row would not do, since those rows may hold infinities or NaN.  Experts
// without rows get a zero dw, rows outside every expert a zero dx.
//
// Few tiles with a long contraction are cut along it (splits_of), those of a weight gradient are not: one
// expert of 512 x 512 with 20000 rows takes eight tiles and 87 us.
//
// Warps: 0 TMA producer, whose copies complete on the leader's stage barrier; 1 MMA issuer
// (leader CTA); 2 clears the tail of a segment's last stage (whose copies complete on a barrier
// of its own CTA) and hands it to the leader; 4-11 epilogue, eight warps of 32 rows x 128 columns.
// Measured and not kept: sixteen epilogue warps (dw of 12288 rows on 64 experts 128 us against
// 123; both before whole blocks left by tiled stores, not measured again), 64 contraction values a
// stage (six stages: the same within 2 % for whole tiles, 21 against 18.8 us for dx of 1024 rows in
// 128-column tiles).
//
// An accumulator holds a whole contraction (or range of it) in fp32, and the tensor pipe truncates
// where it adds: sums of one sign come out low, by 8e-7 of their value after 1024 bf16 products of
// mean 1, 2.5e-5 after 8192, 3.4e-4 after 65536; random signs are off by 1e-5 (rms) after 8192.  That
// is below half a step of bf16 up to some 300 000 products, of fp16 up to some 40 000; fp32 weight
// gradients show it.  (fp32 operands, grad_split.cu, are summed 64 products at a time for that reason.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "grad_tile.cuh"

namespace lmoe {
namespace {

constexpr int kSK = 128;           // contraction values per stage
constexpr int kStages = 3, kAcc = 2;
constexpr int kEpiWarp0 = 4, kEpiWarps = 8;
constexpr int kThreads = (kEpiWarp0 + kEpiWarps) * 32;
constexpr uint32_t kChunk = kSK * 128;            // 128 contraction rows of 64 columns, or 128 rows
                                                  // of 64 contraction values
constexpr uint32_t kOperand = 2 * kChunk;         // 128 x 128 values of one operand
constexpr uint32_t kStageBytes = 2 * kOperand;
constexpr uint32_t kBlockBytes = 32 * 128;        // a warp's block on its way out
constexpr uint32_t kSite = 0x900u;

struct __align__(8) Bars {
  uint64_t full[kStages];       // leader: both CTAs' operands landed (one arrival each)
  uint64_t empty[kStages];      // the stage's MMAs finished (both CTAs)
  uint64_t tail[kStages];       // this CTA's operands of a stage with a tail to clear
  uint64_t acc_full[kAcc];
  uint64_t acc_empty[kAcc];     // leader: both CTAs' epilogue warps
  uint64_t mma_done;
  uint32_t tmem_base;
  int abort;
  SegTable seg;
};

// The part of a tile that unit `unit` sums: one of a.splits ranges of its stages, from k0 on.
struct Part {
  Tile t;
  int k0, s;
};
template <int FORM>
__device__ __forceinline__ Part part_at(const SegTable& seg, const GradArgs& a, int unit, int& hint) {
  Part p;
  p.k0 = p.s = 0;
  if (FORM != kGradWeight && a.splits > 1) {
    p.s = unit % a.splits;
    unit /= a.splits;
  }
  p.t = tile_at<FORM, kSK>(seg, a, unit, hint);
  if (FORM != kGradWeight && a.splits > 1) {
    p.k0 = p.t.ks * p.s / a.splits;
    p.t.ks = p.t.ks * (p.s + 1) / a.splits - p.k0;
  }
  return p;
}

// Whether a stage with `left` rows of its segment ends inside the 16 rows of an MMA.
__device__ __forceinline__ bool has_tail(int left) { return left < kSK && (left & 15) != 0; }

template <int FORM>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    grad_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_a32,
                     const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_out,
                     const GradArgs a) {
  extern __shared__ __align__(1024) uint8_t base[];   // whole swizzle atoms
  uint8_t* store_stage = base + kStages * kStageBytes;
  Bars* bars = reinterpret_cast<Bars*>(store_stage + kEpiWarps * kBlockBytes);
  volatile int* abort_flag = &bars->abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars->full[s], 2);
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
  load_segments(&bars->seg, a.offsets, a.offsets_i64, a.E, a.R, tid, kThreads);
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
  const int total = seg.tile_start[segs] * (FORM != kGradWeight ? a.splits : 1);
  const int first = blockIdx.x >> 1, stride = gridDim.x >> 1;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    const uint32_t full_addr = mapa_u32(&bars->full[0], 0);
    Ring<kStages> st;
    int hint = 0;
    bool ok = true;
    for (int tile = first; tile < total && ok; tile += stride) {
      const Part part = part_at<FORM>(seg, a, tile, hint);
      const Tile& t = part.t;
      const int c0 = t.n * a.width + (int)rank * (a.width / 2);   // first column of B
      const int m0 = (FORM != kGradWeight ? t.row0 : t.m * kTile) + (int)rank * kCta;
      int boxes = 4;   // input gradient: 32-row boxes of dy that hold this CTA's rows
      if (FORM != kGradWeight) {
        const int rows = t.row_end - m0;
        boxes = rows <= 0 ? 0 : (rows >= kCta ? 4 : (rows + 31) >> 5);
      }
      const bool wide = a.width == kTile;
      const uint32_t b_bytes = wide ? kOperand : kChunk;
      for (int i = 0; i < t.ks; ++i, st.next()) {
        const int ks = part.k0 + i;
        ok = warp_wait(&bars->empty[st.i], st.phase ^ 1u, a.err, abort_flag, kSite + 2);
        if (!ok) break;
        if (elect_one()) {
          uint8_t* sa = base + st.i * kStageBytes;
          uint8_t* sb = sa + kOperand;
          const uint32_t bar = full_addr + st.i * 8;
          if (FORM != kGradWeight) {
            const int blocks = a.N - ks * kSK > 64 ? 2 : 1;
            const uint32_t b_block = (uint32_t)a.width * 64u;   // product: width / 2 rows of 64 values
            mbar_arrive_expect_tx_cluster(
                bar, (uint32_t)(blocks * boxes) * 4096u + (FORM == kGradProduct ? blocks * b_block : b_bytes));
            for (int h = 0; h < blocks; ++h) {
              const int x = ks * kSK + h * 64;
              if (boxes == 4) {
                tma_load_2d_pair(sa + h * kChunk, &tm_a, bar, x, m0);
              } else {
                for (int b = 0; b < boxes; ++b)
                  tma_load_2d_pair(sa + h * kChunk + b * 4096, &tm_a32, bar, x, m0 + b * 32);
              }
            }
            if (FORM == kGradProduct) {
              for (int h = 0; h < blocks; ++h)
                tma_load_3d_pair(sb + h * b_block, &tm_b, bar, ks * kSK + h * 64, c0, t.e);
            } else {
              tma_load_3d_pair(sb, &tm_b, bar, c0, ks * kSK, t.e);
              if (wide) tma_load_3d_pair(sb + kChunk, &tm_b, bar, c0 + 64, ks * kSK, t.e);
            }
          } else {
            const int r = t.row0 + ks * kSK;
            const int left = t.row_end - r;
            const int halves = left > 64 ? 2 : 1;   // 64-row boxes that hold rows of the segment
            const uint32_t bytes = (uint32_t)halves * (kOperand + b_bytes) / 2;
            if (has_tail(left)) {
              uint64_t* own = &bars->tail[st.i];
              mbar_arrive_expect_tx(own, bytes);
              for (int h = 0; h < halves; ++h) {
                uint8_t *da = sa + h * (kChunk / 2), *db = sb + h * (kChunk / 2);
                tma_load_2d(da, &tm_a, own, m0, r + h * 64);
                tma_load_2d(da + kChunk, &tm_a, own, m0 + 64, r + h * 64);
                tma_load_2d(db, &tm_b, own, c0, r + h * 64);
                if (wide) tma_load_2d(db + kChunk, &tm_b, own, c0 + 64, r + h * 64);
              }
            } else {
              mbar_arrive_expect_tx_cluster(bar, bytes);
              for (int h = 0; h < halves; ++h) {
                uint8_t *da = sa + h * (kChunk / 2), *db = sb + h * (kChunk / 2);
                tma_load_2d_pair(da, &tm_a, bar, m0, r + h * 64);
                tma_load_2d_pair(da + kChunk, &tm_a, bar, m0 + 64, r + h * 64);
                tma_load_2d_pair(db, &tm_b, bar, c0, r + h * 64);
                if (wide) tma_load_2d_pair(db + kChunk, &tm_b, bar, c0 + 64, r + h * 64);
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
      const uint32_t idesc = idesc_f16kind_f32(kTile, a.width, a.f16) | (FORM == kGradProduct ? 0u : kIdescBMajorMN) |
                             (FORM == kGradWeight ? kIdescAMajorMN : 0u);
      // descriptors count 16 bytes
      const uint64_t adesc0 = FORM != kGradWeight ? sdesc_k_sw128(smem_u32(base)) : sdesc_mn_sw128(smem_u32(base), kChunk);
      const uint64_t bdesc0 = FORM == kGradProduct ? sdesc_k_sw128(smem_u32(base) + kOperand)
                                               : sdesc_mn_sw128(smem_u32(base) + kOperand, kChunk);
      const uint32_t b_step = (uint32_t)a.width * 4u;   // product: the next 64 contraction values
      Ring<kStages> st;
      Ring<kAcc> ac;
      int hint = 0;
      bool ok = true;
      for (int tile = first; tile < total && ok; tile += stride) {
        const Part part = part_at<FORM>(seg, a, tile, hint);
        const Tile& t = part.t;
        const int depth = FORM != kGradWeight ? a.N : t.row_end - t.row0;
        if (t.ks != 0) {
          ok = warp_wait(&bars->acc_empty[ac.i], ac.phase ^ 1u, a.err, abort_flag, kSite + 4);
          if (!ok) break;
          const uint32_t d = tmem + ac.i * kTile;
          for (int ks = 0; ks < t.ks; ++ks, st.next()) {
            ok = warp_wait(&bars->full[st.i], st.phase, a.err, abort_flag, kSite + 6);
            if (!ok) break;
            tc_fence_after();
            const int left = depth - (part.k0 + ks) * kSK;
            if (elect_one()) {
              const uint64_t ad = adesc0 + st.i * (kStageBytes >> 4), bd = bdesc0 + st.i * (kStageBytes >> 4);
#pragma unroll
              for (int kk = 0; kk < kSK / 16; ++kk) {
                // 16 contraction values: 32 bytes of the lines of a K-major block, or 16 lines
                const uint32_t step = FORM != kGradWeight ? (kk >> 2) * (kChunk >> 4) + (kk & 3) * 2 : kk * 128;
                const uint32_t bstep = FORM == kGradProduct ? (kk >> 2) * b_step + (kk & 3) * 2 : kk * 128;
                if (kk * 16 < left) mma_ss_pair(d, ad + step, bd + bstep, idesc, (ks | kk) != 0 ? 1u : 0u);
              }
              mma_commit_pair(&bars->empty[st.i]);
              if (ks == t.ks - 1) mma_commit_pair(&bars->acc_full[ac.i]);
            }
            __syncwarp();
          }
          ac.next();
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
        for (int ks = 0; ks < t.ks && ok; ++ks, st.next()) {
          if (ks != t.ks - 1 || !has_tail(left)) continue;
          ok = warp_wait(&bars->tail[st.i], tail_parity >> st.i & 1u, a.err, abort_flag, kSite + 8);
          if (!ok) break;
          tail_parity ^= 1u << st.i;
          // contraction rows [left, next multiple of 16) of the four chunks; a row is one
          // 128-byte line, which the swizzle only permutes
          const int m = (16 - (left & 15)) * 8;
          uint8_t* at = base + st.i * kStageBytes + left * 128;
          for (int k = lane; k < 4 * m; k += 32) {
            const int c = k / m;
            *reinterpret_cast<uint4*>(at + c * kChunk + (k - c * m) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_u32(&bars->full[st.i], 0));
        }
      }
    }
  } else if (warp >= kEpiWarp0) {
    // ------------------------------------------------------------------ epilogue
    const int q = warp & 3, half = (warp - kEpiWarp0) >> 2;
    const uint32_t lane_base = (uint32_t)(q * 32) << 16;
    const uint32_t empty_addr = mapa_u32(&bars->acc_empty[0], 0);
    const int odt = a.out_dtype;
    const int64_t pitch = (int64_t)a.K * (odt == LMOE_DTYPE_F32 ? 4 : 2);
    uint8_t* stage = store_stage + (warp - kEpiWarp0) * kBlockBytes;
    Ring<kAcc> ac;
    int hint = 0;
    bool ok = true;
    for (int tile = first; tile < total; tile += stride) {
      const Part part = part_at<FORM>(seg, a, tile, hint);
      const Tile& t = part.t;
      // the warp's 32 rows, and the first of its half of the columns
      const int r = (int)rank * kCta + q * 32;
      const int left = FORM != kGradWeight ? t.row_end - t.row0 - r : a.N - t.m * kTile - r;
      const int rows = left < 32 ? left : 32;
      const int64_t row = FORM != kGradWeight ? part.s * a.R + t.row0 + r : (int64_t)t.e * a.N + t.m * kTile + r;
      uint8_t* out = static_cast<uint8_t*>(a.out) + row * pitch;
      const int cols = a.width / 2;
      const int c0 = t.n * a.width + half * cols;
      const uint32_t col0 = tmem + lane_base + half * cols;
      // whole 32-row blocks leave by TMA; a weight gradient's rows behind N are cut by the tensor map
      const bool whole = a.store != kStoreStaged && (FORM == kGradWeight ? rows > 0 : rows == 32);
      const int y = FORM == kGradWeight ? t.m * kTile + r : t.row0 + r, z = FORM == kGradWeight ? t.e : part.s;
      if (t.ks != 0) {
        ok = warp_wait(&bars->acc_full[ac.i], ac.phase, a.err, abort_flag, kSite + 9);
        if (!ok) break;
        tc_fence_after();
      }
      for (int j = 0; j < cols; j += 64) {
        float f[64];
        if (t.ks != 0) {
          uint32_t u[32], v[32];
          tmem_ld32x2(col0 + ac.i * kTile + j, col0 + ac.i * kTile + j + 32, u, v);
          if (j + 64 == cols) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(empty_addr + ac.i * 8);
            ac.next();
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            f[i] = __uint_as_float(u[i]);
            f[32 + i] = __uint_as_float(v[i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 64; ++i) f[i] = 0.0f;
        }
        const int c = c0 + j;
        if (c >= a.K) continue;
        if (whole && odt != LMOE_DTYPE_F32) {
          store_block<128>(&tm_out, f, odt, stage, lane, c, y, z);
        } else if (whole) {
          store_block<128>(&tm_out, f, odt, stage, lane, c, y, z);
          if (c + 32 < a.K) store_block<128>(&tm_out, f + 32, odt, stage, lane, c + 32, y, z);
        } else {
          store_rows<64, kBlockBytes>(out, pitch, rows, c, a.K, f, odt, a.store, stage, lane);
        }
      }
    }
    if (elect_one()) bulk_wait_all();   // the stores are complete
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();   // the other CTA's arrivals and the MMAs on this CTA's memory are done
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// dst[r, 0 .. pitch) = src[r, 0 .. cols) and zeros: 16-bit rows whose length is not a multiple of
// 16 bytes cannot be read by TMA where they lie.  Rows start at any even address: a thread reads
// the five aligned words around its eight values and shifts them into place (value by value, 8
// loads, the copies of 11147 x 6965 values took three times as long).
__global__ void __launch_bounds__(256) pad_rows_kernel(const __grid_constant__ CopyJobs jobs) {
  const CopyJob& job = jobs.job[blockIdx.y];
  const uint16_t* __restrict__ src = static_cast<const uint16_t*>(job.src);
  const int64_t rows = job.rows;
  const int cols = job.cols, pitch = job.pitch;
  uint4* __restrict__ dst = job.dst;
  const int per = pitch / 8;
  const int64_t total = rows * per;
  const int head = (int)(reinterpret_cast<uintptr_t>(src) >> 1 & 1);   // values of the first word before src
  const uint16_t* base = src - head;
  const int64_t end = rows * cols + head;   // values from base
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / per;
    const int c = (int)(i - r * per) * 8;
    const int64_t at = r * cols + c + head, x = at & ~int64_t(1);
    uint32_t w[5];
    if (x >= head && x + 10 <= end) {
#pragma unroll
      for (int j = 0; j < 5; ++j) w[j] = __ldg(reinterpret_cast<const uint32_t*>(base + x) + j);
    } else {   // the ends of src: values that are its own
#pragma unroll
      for (int j = 0; j < 5; ++j) {
        const int64_t k = x + 2 * j;
        w[j] = (k >= head && k < end ? __ldg(base + k) : 0u) | (k + 1 < end ? (uint32_t)__ldg(base + k + 1) << 16 : 0u);
      }
    }
    uint32_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = (at & 1) ? __funnelshift_r(w[j], w[j + 1], 16) : w[j];
      const int left = cols - c - 2 * j;   // values of the row from here on
      if (left < 2) v[j] = left == 1 ? v[j] & 0xffffu : 0u;
    }
    dst[i] = make_uint4(v[0], v[1], v[2], v[3]);
  }
}

// out[i] = the sum of part[s][i] over s, in its order; 16-bit values.
__global__ void __launch_bounds__(256) join_kernel(const float* __restrict__ part, int splits, int64_t n, int f16,
                                                   uint16_t* __restrict__ out) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    float v = part[i];
    for (int s = 1; s < splits; ++s) v += part[s * n + i];
    out[i] = (uint16_t)pack16(v, 0.0f, f16);
  }
}

// Ranges that the contraction is summed in where few tiles (of 128 columns) would leave most pairs
// idle, at least four stages each: their fp32 sums go to the workspace and are joined in order (both
// gradients of 5 rows, N = 7680, K = 856: 28 us, were 42).
constexpr int kPairs = 74;   // of a B200
inline int splits_of(const GradProblem& p) {
  if (weight_grad(p) || p.total_rows == 0) return 1;
  const int64_t tiles = even_row_tiles(p.total_rows, p.num_experts, kTile) * ((p.K + 127) / 128);
  const int64_t most = ((int64_t)p.N + kSK - 1) / kSK / 4, fit = kPairs / tiles;
  return (int)(fit < most ? (fit < 1 ? 1 : fit) : (most < 1 ? 1 : most));
}
inline size_t copies_bytes(const GradProblem& p) {
  size_t b = 0;
  if (p.N % 8) b += align256((size_t)p.total_rows * pitch8(p.N) * 2);
  if (other_cols(p) % 8) b += align256((size_t)other_rows(p) * pitch8(other_cols(p)) * 2);
  return b;
}

template <int FORM>
int launch(const CUtensorMap& ta, const CUtensorMap& ta32, const CUtensorMap& tb, const CUtensorMap& to,
           const GradArgs& a, int grid, cudaStream_t stream) {
  constexpr size_t smem = kStages * kStageBytes + kEpiWarps * kBlockBytes + sizeof(Bars);
  static_assert(smem <= 232448, "shared memory budget");
  auto fn = grad_gemm_kernel<FORM>;
  const int st = set_max_dynamic_smem(reinterpret_cast<const void*>(fn), smem);
  if (st != LMOE_OK) return st;
  fn<<<grid, kThreads, smem, stream>>>(ta, ta32, tb, to, a);
  return cuda_status(cudaGetLastError());
}

}  // namespace

size_t grad_gemm_workspace(const GradProblem& p) {
  if (p.dtype == LMOE_DTYPE_F32) return grad_split_workspace(p);
  const int splits = splits_of(p);
  return copies_bytes(p) + (splits > 1 ? (size_t)splits * p.total_rows * p.K * 4 : 0);
}
size_t grad_gemm_needs(const GradProblem& p) {
  return p.dtype == LMOE_DTYPE_F32 ? grad_split_workspace(p) : copies_bytes(p);
}

int run_grad_gemm(const GradProblem& p, cudaStream_t stream) {
  DeviceInfo dev;
  int st = get_device_info(&dev);
  if (st != LMOE_OK) return st;
  if (dev.cc_major != 10) return LMOE_ERR_DEVICE;
  const void* dy = p.dy;
  const void* other = p.other;
  const int64_t ldy = pitch8(p.N), ldo = pitch8(other_cols(p));
  uint8_t* ws = static_cast<uint8_t*>(p.workspace);
  CopyJobs jobs = {};
  if (ldy != p.N) {
    jobs.add(p.dy, p.total_rows, p.N, ldy, ws);
    dy = ws;
    ws += align256((size_t)p.total_rows * ldy * 2);
  }
  if (ldo != other_cols(p)) {
    jobs.add(p.other, other_rows(p), other_cols(p), ldo, ws);
    other = ws;
    ws += align256((size_t)other_rows(p) * ldo * 2);
  }
  if (jobs.count) {
    pad_rows_kernel<<<jobs.grid(dev), 256, 0, stream>>>(jobs);
    st = cuda_status(cudaGetLastError());
    if (st != LMOE_OK) return st;
  }
  GradArgs a = {};
  CUtensorMap ta, ta32, tb, to = {};
  int splits = splits_of(p);
  if (p.workspace_bytes < grad_gemm_workspace(p)) splits = 1;
  GradProblem q = p;
  if (splits > 1) {   // the sums of the ranges: splits matrices like the output, in fp32
    q.out = ws;
    q.out_dtype = LMOE_DTYPE_F32;
  }
  st = fill_args(q, kSK, splits, a, to);
  if (st != LMOE_OK) return st;
  const CUtensorMapDataType dt = a.f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const int grid = gemm_grid(dev) < 2 ? 2 : gemm_grid(dev) & ~1;   // whole pairs
  const int64_t row_tiles = weight_grad(p) ? (int64_t)a.MT * p.num_experts
                                          : even_row_tiles(p.total_rows, p.num_experts, kTile);
  const int widths[] = {256, 128};
  a.width = splits > 1 ? 128 : pick_width(widths, grid / 2, 0, 16, [&](int w) { return row_tiles * ((p.K + w - 1) / w); });
  a.raster = Raster((p.K + a.width - 1) / a.width);
  // the maps end at the true sizes, so that TMA fills what lies behind them with zeros
  if (weight_grad(p)) {
    st = encode_tmap_2d(&ta, dy, dt, 2, (uint64_t)p.total_rows, (uint64_t)p.N, (uint64_t)ldy * 2, 64, 64, true);
    if (st != LMOE_OK) return st;
    st = encode_tmap_2d(&tb, other, dt, 2, (uint64_t)p.total_rows, (uint64_t)p.K, (uint64_t)ldo * 2, 64, 64, true);
    if (st != LMOE_OK) return st;
    return launch<kGradWeight>(ta, ta, tb, to, a, grid, stream);
  }
  st = encode_tmap_2d(&ta, dy, dt, 2, (uint64_t)p.total_rows, (uint64_t)p.N, (uint64_t)ldy * 2, kCta, 64, true);
  if (st != LMOE_OK) return st;
  st = encode_tmap_2d(&ta32, dy, dt, 2, (uint64_t)p.total_rows, (uint64_t)p.N, (uint64_t)ldy * 2, 32, 64, true);
  if (st != LMOE_OK) return st;
  const bool product = p.form == kGradProduct;
  const uint64_t rows = (uint64_t)(product ? p.K : p.N);   // of one expert's matrix
  const uint64_t dims[3] = {(uint64_t)other_cols(p), rows, (uint64_t)p.num_experts};
  const uint64_t strides[2] = {(uint64_t)ldo * 2, (uint64_t)ldo * 2 * rows};
  const uint32_t box[3] = {64, product ? (uint32_t)a.width / 2 : (uint32_t)kSK, 1};
  st = encode_tmap_3d(&tb, other, dt, 2, dims, strides, box);
  if (st != LMOE_OK) return st;
  st = product ? launch<kGradProduct>(ta, ta32, tb, to, a, grid, stream)
               : launch<kGradInput>(ta, ta32, tb, to, a, grid, stream);
  if (st != LMOE_OK || splits == 1) return st;
  const int64_t n = p.total_rows * p.K, blocks = (n + 255) / 256, enough = (int64_t)dev.num_sms * 8;
  join_kernel<<<(unsigned)(blocks < enough ? blocks : enough), 256, 0, stream>>>(
      static_cast<const float*>(q.out), splits, n, a.f16, static_cast<uint16_t*>(p.out));
  return cuda_status(cudaGetLastError());
}

}  // namespace lmoe

using namespace lmoe;

namespace {

int grad_entry(GradProblem& p, const void* offsets, void* out, void* workspace, size_t workspace_bytes,
               cudaStream_t stream) {
  LMOE_ARG_CHECK(p.dtype == LMOE_DTYPE_BF16 || p.dtype == LMOE_DTYPE_F16 || p.dtype == LMOE_DTYPE_F32);
  LMOE_ARG_CHECK(p.out_dtype == p.dtype || (weight_grad(p) && p.out_dtype == LMOE_DTYPE_F32));
  LMOE_ARG_CHECK(p.total_rows >= 0 && p.N > 0 && p.K > 0 && p.num_experts >= 1);
  // indexes of whole tiles and stages stay within 32 bits
  LMOE_ARG_CHECK(p.total_rows <= kMaxGemmSize && p.N <= kMaxGemmSize && p.K <= kMaxGemmSize);
  if (p.num_experts > kMaxGemmExperts) return LMOE_ERR_UNSUPPORTED;
  const int64_t esize = p.dtype == LMOE_DTYPE_F32 ? 4 : 2, osize = p.out_dtype == LMOE_DTYPE_F32 ? 4 : 2;
  LMOE_ARG_CHECK(out && reinterpret_cast<uintptr_t>(out) % osize == 0);
  if (p.total_rows == 0) {
    if (!weight_grad(p)) return LMOE_OK;
    return cuda_status(cudaMemsetAsync(out, 0, (size_t)p.num_experts * p.N * p.K * osize, stream));
  }
  LMOE_ARG_CHECK(p.dy && p.other && offsets);
  LMOE_ARG_CHECK(reinterpret_cast<uintptr_t>(p.dy) % esize == 0 && reinterpret_cast<uintptr_t>(p.other) % esize == 0);
  if (p.dtype == LMOE_DTYPE_F32 && (!workspace || !grad_splits(p))) return run_grad_f32(p, stream);
  // rows that TMA reads where they lie start at multiples of 16 bytes
  LMOE_ARG_CHECK(p.dtype == LMOE_DTYPE_F32 ||
                 ((p.N % 8 || aligned16(p.dy)) && (other_cols(p) % 8 || aligned16(p.other))));
  const size_t need = grad_gemm_needs(p);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return LMOE_ERR_WORKSPACE;
  p.workspace = workspace;
  p.workspace_bytes = workspace && aligned16(workspace) ? workspace_bytes : 0;
  return p.dtype == LMOE_DTYPE_F32 ? run_grad_split(p, stream) : run_grad_gemm(p, stream);
}

}  // namespace

extern "C" size_t lmoe_grouped_gemm_grad_workspace_bytes(int form, int dtype, int64_t total_rows, int N, int K,
                                                         int num_experts) {
  if (form < 0 || form > 2 || total_rows < 0 || N <= 0 || K <= 0 || num_experts <= 0) return 0;
  if (total_rows > kMaxGemmSize || N > kMaxGemmSize || K > kMaxGemmSize) return 0;   // refused
  GradProblem p;
  p.form = form;
  p.dtype = dtype;
  p.total_rows = total_rows;
  p.N = form == kGradProduct ? K : N;   // contraction and columns
  p.K = form == kGradProduct ? N : K;
  p.num_experts = num_experts;
  return grad_gemm_workspace(p);
}

extern "C" int lmoe_grouped_gemm_dgrad(const void* grad_output, int dtype, int64_t total_rows, int N,
                                       const void* weights, int K, const void* expert_offsets, int offsets_are_int64,
                                       int num_experts, void* grad_input, void* workspace, size_t workspace_bytes,
                                       uint32_t* error, lmoe_stream_t stream) {
  GradProblem p;
  p.form = kGradInput;
  p.dtype = p.out_dtype = dtype;
  p.total_rows = total_rows;
  p.N = N;
  p.K = K;
  p.num_experts = num_experts;
  p.dy = grad_output;
  p.other = weights;
  p.offsets = expert_offsets;
  p.offsets_i64 = offsets_are_int64;
  p.out = grad_input;
  p.err = error;
  if (total_rows == 0 && !grad_input) return N > 0 && K > 0 && num_experts >= 1 ? LMOE_OK : LMOE_ERR_INVALID_ARG;
  return grad_entry(p, expert_offsets, grad_input, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int lmoe_grouped_gemm_wgrad(const void* grad_output, int dtype, int64_t total_rows, int N,
                                       const void* input, int K, const void* expert_offsets, int offsets_are_int64,
                                       int num_experts, int out_dtype, void* grad_weights, void* workspace,
                                       size_t workspace_bytes, uint32_t* error, lmoe_stream_t stream) {
  GradProblem p;
  p.form = kGradWeight;
  p.dtype = dtype;
  p.out_dtype = out_dtype;
  p.total_rows = total_rows;
  p.N = N;
  p.K = K;
  p.num_experts = num_experts;
  p.dy = grad_output;
  p.other = input;
  p.offsets = expert_offsets;
  p.offsets_i64 = offsets_are_int64;
  p.out = grad_weights;
  p.err = error;
  return grad_entry(p, expert_offsets, grad_weights, workspace, workspace_bytes,
                    reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int lmoe_grouped_gemm_any(const void* input, int dtype, int64_t total_rows, int K, const void* weights, int N,
                                     const void* expert_offsets, int offsets_are_int64, int num_experts, void* output,
                                     void* workspace, size_t workspace_bytes, uint32_t* error, lmoe_stream_t stream) {
  GradProblem p;
  p.form = kGradProduct;
  p.dtype = p.out_dtype = dtype;
  p.total_rows = total_rows;
  p.N = K;
  p.K = N;
  p.num_experts = num_experts;
  p.dy = input;
  p.other = weights;
  p.offsets = expert_offsets;
  p.offsets_i64 = offsets_are_int64;
  p.out = output;
  p.err = error;
  if (total_rows == 0 && !output) return N > 0 && K > 0 && num_experts >= 1 ? LMOE_OK : LMOE_ERR_INVALID_ARG;
  return grad_entry(p, expert_offsets, output, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}
