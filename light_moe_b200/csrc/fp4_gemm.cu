// fp4_gemm.cu -- grouped product of microscaled 4-bit operands on CTA pairs (sm_100a).
//
//   y[r, n] = alpha[e] * sum_k x[r, k] * w[e, n, k]      for the rows r of expert e
//   y[r, f] = silu(gate[r, f]) * up[r, f]                with a gate and an up matrix
//
// Both operands are E2M1 with a scale byte per 32 (MX) or 16 (NV) values (fp4_format.cuh); the
// block-scaled tcgen05.mma multiplies codes and scales exactly and accumulates in fp32, four
// times the bf16 rate for a quarter of the bytes.  With few rows the weights' bytes bound it (HBM).
// With many, a long run of calls is bound by power (8 experts of 2 x 14336 x 4096, 700 rows each: 373 us at
// the 1327 MHz that 1000 W leave), a single call by no one part: 310 us at 1965 MHz, 153 of them MMAs;
// with half of the codes' copies 285, without the loads of the scales too 256, without the copies
// of the scales to tensor memory 309, without the stores ~295.
//
// Tile: 256 rows (128 per CTA, TMEM lane = row) x 192 weight rows (96 per CTA in shared memory).
// (Narrower tiles for a fuller last round measured slower from 64 rows per expert on: 119 against
// 112 us for 8 experts of 2 x 14336 x 4096.)
// 192 columns because two accumulators (2 x 192) and two buffers of scales (2 x 48 columns) fit
// the 512 TMEM columns, so the epilogue of a tile overlaps the next tile's MMAs; 256 columns
// would leave room for one accumulator only.  The lane being the row, a thread holds a row's
// gate and up values of the same features, and the SwiGLU needs no exchange: for gate / up the
// leader's 96 columns are gate rows and the follower's 96 the same rows of up.
//
// Operands stay in the canonical layout of the quantiser (codes [rows, K/2], scales [rows,
// pitch]): the codes arrive by TMA (128-byte swizzle, 256 values = 128 bytes a row), two such blocks a stage.
// The scales must lie in shared memory as 512-byte tiles of 128 rows x 4 scales, row r at
// (r % 32) * 16 + (r / 32) * 4, from where tcgen05.cp copies them to TMEM.  Five warps of 64 rows
// each read them as whole 32-byte sectors a row (a step: the scales of two stages of MX, one of
// NV), three steps ahead in registers, write the tiles and hand a step to the leader in one go.
//
// One thread issues a unit of four 4-scale words a row (512 values of MX, 256 of NV: twelve copies
// into one of two TMEM buffers of 48 columns) and its MMAs, in whose order the tensor pipe runs
// them.  A wait costs it ~65 cycles and an instruction ~25, against 96 cycles an MMA; so a stage holds
// 512 values and the waits of a unit start together.  (With 256 values and one wait after another:
// 650 cycles per 384 of MMAs, 0.88 ms for the gate / up product of 16384 rows, now 0.79; with the
// copies issued by a warp of their own they queue behind the MMAs issued before, and the hand-over
// then stands in the pipe.)
//
// Warps: 0 TMA producer, whose copies complete on the leader's stage barrier; 1 MMA issuer
// (leader CTA); 2-3 scales of the rows, 4-6 scales of the 192 columns (each CTA keeps all: the MMA
// reads them beside its own rows); from 7 on the epilogue: eight warps of 32 rows x 96 columns, or
// twelve of 32 rows x 32 features for the SwiGLU, whose arithmetic wants more warps.  Whole blocks
// of 32 rows x 64 bytes (SwiGLU 32) leave by tiled stores; lanes that store rows of their own kept
// the L1 data pipe busy (64 experts of 2048 x 1408, 700 rows each: 100 us, was 134).  With eight
// warps the SwiGLU of 64 experts of 2 x 1408 x 2048 takes 163 us, with twelve 139.
#include <cuda_bf16.h>

#include "fp4_mma.cuh"
#include "host_util.h"

namespace lmoe {
namespace {

constexpr int kRowsCta = 128, kTM = 256, kTN = 192, kHalf = 96;
constexpr int kBK = kFp4Block, kSK = kFp4Stage;
constexpr int kStages = 3, kAcc = 2;
constexpr int kSfSlots = 3;       // steps of scales in shared memory
constexpr int kUnits = 2;         // units of scales in TMEM
constexpr uint32_t kUnitCols = 48;   // 4 words x (4 columns of the rows' scales, 8 of the columns')
constexpr int kSfWarp0 = 2, kSfWarps = 5, kEpiWarp0 = 7;
// The epilogue's warps: SwiGLU twelve of 32 features, a product eight of 96 columns.
template <bool SWIGLU>
struct Epi {
  static constexpr int kWarps = SWIGLU ? 12 : 8, kThreads = (kEpiWarp0 + kWarps) * 32;
  static constexpr int kCols = SWIGLU ? 16 : 32, kBlocks = SWIGLU ? 2 : 3;   // of a block; blocks a warp
  static constexpr uint32_t kBlockBytes = 32 * kCols * 2;                   // a block on its way out
};
constexpr uint32_t kABlock = kRowsCta * 128, kBBlock = kHalf * 128;
constexpr uint32_t kABytes = 2 * kABlock, kBBytes = 2 * kBBlock;
constexpr uint32_t kSite = 0x500u;
constexpr int kTmemCols = 512;
struct __align__(8) Bars {
  uint64_t full[kStages];       // leader: both CTAs' codes landed (one arrival each)
  uint64_t empty[kStages];      // the stage's MMAs finished (both CTAs)
  uint64_t sf_full[kSfSlots];   // leader: both CTAs' scale warps wrote the step
  uint64_t sf_empty[kSfSlots];  // the step's scales were copied (both CTAs)
  uint64_t unit_empty[kUnits];  // leader: the unit's MMAs finished
  uint64_t acc_full[kAcc];
  uint64_t acc_empty[kAcc];     // leader: both CTAs' epilogue warps
  uint64_t mma_done;
  uint32_t tmem_base;
  int abort;
  SegTable seg;
};

static_assert(kAcc * kTN + kUnits * kUnitCols <= kTmemCols, "tensor memory budget");
constexpr uint32_t kStageBytes = kABytes + kBBytes;
constexpr uint32_t kSfABytes = 8 * 512, kSfBBytes = 8 * 1024, kSfSlotBytes = kSfABytes + kSfBBytes;
constexpr uint32_t kEpiBytes = 8 * 2048;   // of the epilogue's blocks (SwiGLU 12 * 1024)
constexpr uint32_t kSmem = 1024 + kStages * kStageBytes + kSfSlots * kSfSlotBytes + kEpiBytes + sizeof(Bars);
static_assert(kStageBytes % 1024 == 0, "swizzle atoms");
static_assert(kSmem <= 232448, "shared memory budget");

template <int FORMAT, bool SWIGLU>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Epi<SWIGLU>::kThreads, 1)
    fp4_gemm_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_x32,
                    const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_up,
                    const __grid_constant__ CUtensorMap tm_out, const Fp4Args a) {
  using C = Fp4Units<FORMAT>;
  using Ep = Epi<SWIGLU>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sf_base = base + kStages * kStageBytes;
  uint8_t* store_stage = sf_base + kSfSlots * kSfSlotBytes;
  Bars* bars = reinterpret_cast<Bars*>(store_stage + kEpiBytes);
  volatile int* abort_flag = &bars->abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars->full[s], 2);
      mbar_init(&bars->empty[s], 1);
    }
    for (int s = 0; s < kSfSlots; ++s) {
      mbar_init(&bars->sf_full[s], 2 * kSfWarps);
      mbar_init(&bars->sf_empty[s], 1);
    }
    for (int s = 0; s < kUnits; ++s) mbar_init(&bars->unit_empty[s], 1);
    for (int s = 0; s < kAcc; ++s) {
      mbar_init(&bars->acc_full[s], 1);
      mbar_init(&bars->acc_empty[s], 2 * Ep::kWarps);
    }
    mbar_init(&bars->mma_done, 1);
    bars->abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(&bars->tmem_base, kTmemCols);
    tmem_relinquish_pair();
  }
  load_segments(&bars->seg, a.offsets, a.offsets_i64, a.E, a.R, tid, Ep::kThreads);
  const int segs = a.E + 2;
  if (warp == 0)
    scan_tiles(&bars->seg, segs, lane, [&](int j) {
      return (bars->seg.row[j + 1] - bars->seg.row[j] + kTM - 1) / kTM * a.raster.nb;
    });
  if (tid == 0 && bars->seg.bad && blockIdx.x == 0) report_error(a.err, kErrBadArg, kSite + 1);
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  const SegTable& seg = bars->seg;
  const int total = seg.tile_start[segs];
  const int KS = a.KS;
  const int first = blockIdx.x >> 1, stride = gridDim.x >> 1;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    const uint32_t full_addr = mapa_u32(&bars->full[0], 0);
    const CUtensorMap* wmap = SWIGLU && !leader ? &tm_up : &tm_w;
    Ring<kStages> st;
    int hint = 0;
    bool ok = true;
    for (int tile = first; tile < total && ok; tile += stride) {
      const Fp4Tile t = fp4_tile_at<kTM>(seg, a, tile, hint);
      if (t.zero) continue;
      const int r0 = t.row0 + (int)rank * kRowsCta;
      int rows = t.row_end - r0;
      rows = rows < 0 ? 0 : (rows > kRowsCta ? kRowsCta : rows);
      const int boxes = (rows + 31) >> 5;   // only the boxes that hold this tile's rows
      const int wrow = SWIGLU ? t.n * kHalf : t.n * kTN + (int)rank * kHalf;
      for (int ks = 0; ks < KS; ++ks, st.next()) {
        ok = warp_wait(&bars->empty[st.i], st.phase ^ 1u, a.err, abort_flag, kSite + 2);
        if (!ok) break;
        if (elect_one()) {
          uint8_t* dst = base + st.i * kStageBytes;
          const uint32_t bar = full_addr + st.i * 8;
          const int blocks = a.K - ks * kSK > kBK ? 2 : 1;
          mbar_arrive_expect_tx_cluster(bar, (uint32_t)blocks * ((uint32_t)boxes * 4096u + kBBlock));
          for (int h = 0; h < blocks; ++h) {
            const int x = ks * (kSK / 2) + h * 128;
            if (boxes == 4) {
              tma_load_2d_pair(dst + h * kABlock, &tm_x, bar, x, r0);
            } else {
              for (int b = 0; b < boxes; ++b)
                tma_load_2d_pair(dst + h * kABlock + b * 4096, &tm_x32, bar, x, r0 + b * 32);
            }
            tma_load_3d_pair(dst + kABytes + h * kBBlock, wmap, bar, x, wrow, t.e);
          }
        }
      }
    }
    // the copies of a finished tile have landed (its MMAs read them)
    if (!ok) let_copies_land();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (leader) {
      const uint64_t adesc0 = sdesc_k_sw128(smem_u32(base)), bdesc0 = sdesc_k_sw128(smem_u32(base) + kABytes);
      const uint64_t sfa0 = sdesc_scales(smem_u32(sf_base)), sfb0 = sdesc_scales(smem_u32(sf_base) + kSfABytes);
      Ring<kStages> st;
      Ring<kSfSlots> sl;
      Ring<kUnits> un;
      Ring<kAcc> ac;
      int hint = 0;
      bool ok = true;
      for (int tile = first; tile < total && ok; tile += stride) {
        const Fp4Tile t = fp4_tile_at<kTM>(seg, a, tile, hint);
        if (t.zero) continue;
        ok = warp_wait(&bars->acc_empty[ac.i], ac.phase ^ 1u, a.err, abort_flag, kSite + 4);
        const uint32_t d = tmem + ac.i * kTN;
        uint32_t accum = 0;
        for (int left = a.K; left > 0 && ok; left -= C::kStepK) {
          // a step: two units, or one at the end of a row
          const uint64_t sa = sfa0 + sl.i * (kSfSlotBytes >> 4), sb = sfb0 + sl.i * (kSfSlotBytes >> 4);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            constexpr int kU = C::kUnitK;
            if (j * kU >= left) break;
            const bool stage_start = j % C::kStageUnits == 0;
            // the waits start together; what has not come yet is waited for below
            const bool w0 = mbar_test(&bars->unit_empty[un.i], un.phase ^ 1u);
            const bool w1 = j > 0 || mbar_test(&bars->sf_full[sl.i], sl.phase);
            const bool w2 = !stage_start || mbar_test(&bars->full[st.i], st.phase);
            if (!(w0 && w1 && w2)) {
              ok = mbar_wait(&bars->unit_empty[un.i], un.phase ^ 1u, a.err, abort_flag, kSite + 5);
              if (ok && j == 0) ok = mbar_wait(&bars->sf_full[sl.i], sl.phase, a.err, abort_flag, kSite + 9);
              if (ok && stage_start) ok = mbar_wait(&bars->full[st.i], st.phase, a.err, abort_flag, kSite + 6);
            }
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const bool last = (j + 1) * kU >= left;   // of the row
            const bool stage_end = (j + 1) % C::kStageUnits == 0 || last;
            if (elect_one()) {
              const uint32_t sfa = tmem + kAcc * kTN + un.i * kUnitCols, sfb = sfa + 16;
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                const int q = 4 * j + w;   // word of the step
                copy_scales_pair(sfa + w * 4, sa + q * 32);
                copy_scales_pair(sfb + w * 8, sb + q * 64);
                copy_scales_pair(sfb + w * 8 + 4, sb + q * 64 + 32);
              }
              // descriptors count 16 bytes; 64 values (an MMA) are 32 bytes of a block's lines
              const uint64_t ad = adesc0 + st.i * (kStageBytes >> 4), bd = bdesc0 + st.i * (kStageBytes >> 4);
#pragma unroll
              for (int m = 0; m < kU / 64; ++m) {
                if (j * kU + m * 64 < left) {
                  const int kk = (j % C::kStageUnits) * (kU / 64) + m;   // of the stage's eight
                  const uint64_t am = ad + (kk >> 2) * (kABlock >> 4) + (kk & 3) * 2;
                  const uint64_t bm = bd + (kk >> 2) * (kBBlock >> 4) + (kk & 3) * 2;
                  if (FORMAT == LMOE_FP4_MX)
                    // a word holds the scales of 128 values: of two MMAs (scale id 0 and 2)
                    mma_fp4_pair<FORMAT>(d, am, bm, idesc_fp4(true, (m & 1) * 2, kTN), sfa + (m >> 1) * 4,
                                         sfb + (m >> 1) * 8, accum | (uint32_t)(m > 0));
                  else
                    mma_fp4_pair<FORMAT>(d, am, bm, idesc_fp4(false, 0, kTN), sfa + m * 4, sfb + m * 8,
                                         accum | (uint32_t)(m > 0));
                }
              }
              mma_commit_leader(&bars->unit_empty[un.i]);
              if (stage_end) mma_commit_pair(&bars->empty[st.i]);
              if (j == 1 || last) mma_commit_pair(&bars->sf_empty[sl.i]);
              if (last) mma_commit_pair(&bars->acc_full[ac.i]);
            }
            __syncwarp();
            accum = 1;
            un.next();
            if (stage_end) st.next();
          }
          sl.next();
        }
        ac.next();
      }
      if (elect_one()) mma_commit_leader(&bars->mma_done);
      mbar_wait(&bars->mma_done, 0, a.err, nullptr, kSite + 7);
    }
  } else if (warp < kEpiWarp0) {
    // ------------------------------------------------------------------ scales
    const int part = warp - kSfWarp0;   // 0, 1: rows 0-63, 64-127; 2, 3, 4: columns 0-63, 64-127, 128-191
    int hint = 0;
    write_scales<FORMAT, kSfSlots>(
        first, total, stride, a.K,
        sf_base + lane * 16 + (part < 2 ? part * 8u : kSfABytes + (part == 4 ? 512u : (uint32_t)(part - 2) * 8u)),
        part < 2 ? 512u : 1024u, kSfSlotBytes, bars->sf_empty, mapa_u32(&bars->sf_full[0], 0), a.err, abort_flag,
        kSite + 8, lane, [&](int tile, const uint8_t* (&p)[2]) {
          const Fp4Tile t = fp4_tile_at<kTM>(seg, a, tile, hint);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            p[i] = nullptr;
            if (part < 2) {
              const int row = t.row0 + (int)rank * kRowsCta + part * 64 + lane + 32 * i;
              if (row < t.row_end) p[i] = a.xs + (int64_t)row * a.xs_pitch;
            } else if (!t.zero) {
              const int c = (part - 2) * 64 + lane + 32 * i;
              const bool up = SWIGLU && c >= kHalf;
              const int n = SWIGLU ? t.n * kHalf + (up ? c - kHalf : c) : t.n * kTN + c;
              if (c < kTN && n < a.N) p[i] = (up ? a.ws_up : a.ws) + ((int64_t)t.e * a.N + n) * a.ws_pitch;
            }
          }
          return !t.zero;
        });
  } else {
    // ------------------------------------------------------------------ epilogue
    const int q = warp & 3, cg = (warp - kEpiWarp0) >> 2;
    const uint32_t lane_base = (uint32_t)(q * 32) << 16;
    const uint32_t empty_addr = mapa_u32(&bars->acc_empty[0], 0);
    const int64_t pitch = (int64_t)a.N * (a.out_dtype == LMOE_DTYPE_F32 ? 4 : 2);
    uint8_t* stage = store_stage + (warp - kEpiWarp0) * Ep::kBlockBytes;
    Ring<kAcc> ac;
    int hint = 0;
    for (int tile = first; tile < total; tile += stride) {
      const Fp4Tile t = fp4_tile_at<kTM>(seg, a, tile, hint);
      const int row = t.row0 + (int)rank * kRowsCta + q * 32;   // the warp's first
      const int rows = t.row_end - row < 32 ? t.row_end - row : 32;
      uint8_t* out = static_cast<uint8_t*>(a.out) + (int64_t)row * pitch;
      const bool whole = rows == 32 && a.store != kStoreStaged;   // blocks leave by TMA
      float al = 1.0f, au = 1.0f;
      if (!t.zero) {
        if (!warp_wait(&bars->acc_full[ac.i], ac.phase, a.err, abort_flag, kSite + 10)) break;
        tc_fence_after();
        if (rows <= 0) {   // the segment ends before this warp's rows
          if (lane == 0) mbar_arrive_cluster(empty_addr + ac.i * 8);
          ac.next();
          continue;
        }
        if (a.alpha) al = __ldg(a.alpha + t.e);
        if (SWIGLU && a.alpha_up) au = __ldg(a.alpha_up + t.e);
      }
      for (int b = cg * Ep::kBlocks; b < (cg + 1) * Ep::kBlocks; ++b) {
        float f[Ep::kCols];
        if (!t.zero) {
          uint32_t u[Ep::kCols], v[Ep::kCols];
          const uint32_t col = tmem + lane_base + ac.i * kTN + b * Ep::kCols;
          if constexpr (SWIGLU)
            tmem_ld16x2(col, col + kHalf, u, v);
          else
            tmem_ld32(col, u);
          if (b == (cg + 1) * Ep::kBlocks - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(empty_addr + ac.i * 8);
            ac.next();
          }
#pragma unroll
          for (int i = 0; i < Ep::kCols; ++i) {
            f[i] = __fmul_rn(__uint_as_float(u[i]), al);
            if (SWIGLU) f[i] = silu(f[i]) * __fmul_rn(__uint_as_float(v[i]), au);
          }
        } else {
#pragma unroll
          for (int i = 0; i < Ep::kCols; ++i) f[i] = 0.0f;
        }
        const int c = t.n * (SWIGLU ? kHalf : kTN) + b * Ep::kCols;
        if (c >= a.N) continue;
        if (!whole) {
          store_rows<Ep::kCols, Ep::kBlockBytes>(out, pitch, rows, c, a.N, f, a.out_dtype, a.store, stage, lane);
        } else {
          store_block<Ep::kCols * 2>(&tm_out, f, a.out_dtype, stage, lane, c, row, 0);
          if (a.out_dtype == LMOE_DTYPE_F32 && c + Ep::kCols / 2 < a.N)
            store_block<Ep::kCols * 2>(&tm_out, f + Ep::kCols / 2, a.out_dtype, stage, lane, c + Ep::kCols / 2, row, 0);
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
    tmem_dealloc_pair(tmem, kTmemCols);
  }
}

template <int FORMAT, bool SWIGLU>
int launch(const CUtensorMap& x, const CUtensorMap& x32, const CUtensorMap& w, const CUtensorMap& up,
           const CUtensorMap& out, const Fp4Args& a, int grid, cudaStream_t stream) {
  auto fn = fp4_gemm_kernel<FORMAT, SWIGLU>;
  const int st = set_max_dynamic_smem(reinterpret_cast<const void*>(fn), kSmem);
  if (st != LMOE_OK) return st;
  fn<<<grid, Epi<SWIGLU>::kThreads, kSmem, stream>>>(x, x32, w, up, out, a);
  return cuda_status(cudaGetLastError());
}

}  // namespace

int run_fp4_gemm(const Fp4Problem& p, cudaStream_t stream) {
  DeviceInfo dev;
  int st = get_device_info(&dev);
  if (st != LMOE_OK) return st;
  if (dev.cc_major != 10) return LMOE_ERR_DEVICE;
  const bool swiglu = p.wq_up != nullptr;
  Fp4Args a = {};
  a.xs = p.xs;
  a.xs_pitch = p.xs_pitch;
  a.ws = p.ws;
  a.ws_up = p.ws_up;
  a.ws_pitch = p.ws_pitch;
  a.offsets = p.offsets;
  a.offsets_i64 = p.offsets_i64;
  a.E = p.num_experts;
  a.N = p.N;
  a.K = p.K;
  a.R = p.total_rows;
  const int grid = gemm_grid(dev) < 2 ? 2 : gemm_grid(dev) & ~1;   // whole pairs
  a.raster = Raster(swiglu ? (p.N + kHalf - 1) / kHalf : (p.N + kTN - 1) / kTN);
  a.KS = (p.K + kSK - 1) / kSK;
  a.alpha = p.alpha;
  a.alpha_up = p.alpha_up;
  a.out = p.out;
  a.out_dtype = p.out_dtype;
  a.store = store_mode(p.out, p.N, p.out_dtype);
  a.err = p.err;
  CUtensorMap tx, tx32, tw, tu, to = {};
  if (a.store != kStoreStaged) {
    st = encode_store_map(&to, p.out, p.out_dtype, (uint64_t)p.N, (uint64_t)p.total_rows, 1, swiglu ? 32 : 64);
    if (st != LMOE_OK) return st;
  }
  const uint64_t kb = (uint64_t)p.K / 2;
  st = encode_tmap_2d(&tx, p.xq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)p.total_rows, kb, kb, kRowsCta, 128, true);
  if (st != LMOE_OK) return st;
  st = encode_tmap_2d(&tx32, p.xq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)p.total_rows, kb, kb, 32, 128, true);
  if (st != LMOE_OK) return st;
  const uint64_t dims[3] = {kb, (uint64_t)p.N, (uint64_t)p.num_experts};
  const uint64_t strides[2] = {kb, kb * (uint64_t)p.N};
  const uint32_t box[3] = {128, (uint32_t)kHalf, 1};
  st = encode_tmap_3d(&tw, p.wq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, dims, strides, box);
  if (st != LMOE_OK) return st;
  tu = tw;
  if (swiglu) {
    st = encode_tmap_3d(&tu, p.wq_up, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, dims, strides, box);
    if (st != LMOE_OK) return st;
  }
  if (p.format == LMOE_FP4_MX)
    return swiglu ? launch<LMOE_FP4_MX, true>(tx, tx32, tw, tu, to, a, grid, stream)
                  : launch<LMOE_FP4_MX, false>(tx, tx32, tw, tu, to, a, grid, stream);
  return swiglu ? launch<LMOE_FP4_NV, true>(tx, tx32, tw, tu, to, a, grid, stream)
                : launch<LMOE_FP4_NV, false>(tx, tx32, tw, tu, to, a, grid, stream);
}

}  // namespace lmoe

using namespace lmoe;

extern "C" int lmoe_fp4_grouped_gemm(const uint8_t* xq, const uint8_t* xs, int64_t xs_pitch, int64_t total_rows, int K,
                                     const uint8_t* wq, const uint8_t* ws, const uint8_t* wq_up, const uint8_t* ws_up,
                                     int64_t ws_pitch, int N, int format, const void* expert_offsets,
                                     int offsets_are_int64, int num_experts, const float* alpha, const float* alpha_up,
                                     int out_dtype, void* output, uint32_t* error, lmoe_stream_t stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  LMOE_ARG_CHECK(format == LMOE_FP4_MX || format == LMOE_FP4_NV);
  LMOE_ARG_CHECK(out_dtype == LMOE_DTYPE_BF16 || out_dtype == LMOE_DTYPE_F16 || out_dtype == LMOE_DTYPE_F32);
  LMOE_ARG_CHECK(total_rows >= 0 && N > 0 && K > 0 && K % 32 == 0);
  // indexes of whole tiles and stages stay within 32 bits
  LMOE_ARG_CHECK(total_rows <= kMaxGemmSize && N <= kMaxGemmSize && K <= kMaxGemmSize);
  LMOE_ARG_CHECK(num_experts >= 1);
  if (num_experts > kMaxGemmExperts) return LMOE_ERR_UNSUPPORTED;
  LMOE_ARG_CHECK((wq_up == nullptr) == (ws_up == nullptr));
  LMOE_ARG_CHECK(xs_pitch % 32 == 0 && ws_pitch % 32 == 0);
  LMOE_ARG_CHECK(xs_pitch >= fp4_scale_pitch(K, format) && ws_pitch >= fp4_scale_pitch(K, format));
  if (total_rows == 0) return LMOE_OK;
  LMOE_ARG_CHECK(xq && xs && wq && ws && expert_offsets && output);
  LMOE_ARG_CHECK(aligned16(xq) && aligned16(wq) && aligned16(wq_up) && aligned32(xs) && aligned32(ws) &&
                 aligned32(ws_up));
  LMOE_ARG_CHECK(reinterpret_cast<uintptr_t>(output) % (out_dtype == LMOE_DTYPE_F32 ? 4 : 2) == 0);
  Fp4Problem p;
  p.xq = xq;
  p.xs = xs;
  p.xs_pitch = xs_pitch;
  p.total_rows = total_rows;
  p.K = K;
  p.wq = wq;
  p.ws = ws;
  p.wq_up = wq_up;
  p.ws_up = ws_up;
  p.ws_pitch = ws_pitch;
  p.N = N;
  p.format = format;
  p.offsets = expert_offsets;
  p.offsets_i64 = offsets_are_int64;
  p.num_experts = num_experts;
  p.alpha = alpha;
  p.alpha_up = alpha_up;
  p.out_dtype = out_dtype;
  p.out = output;
  p.err = error;
  // Few rows: the weights' bytes bound, and tiles of 256 weight rows stream them best (8 experts of
  // 4096 x 14336, us by rows per expert: 1 50 against 68, 64 63 against 72, 96 76 against 73; 64 of
  // 2048 x 1408: 25 against 34, 39 against 37, 54 against 39).  The SwiGLU's exchange between lanes
  // makes up less (8 of 2 x 14336 x 4096: 1 80 against 102, 32 87 against 107, 64 124 against 110; 64
  // of 2 x 1408 x 2048: 38 against 50, 16 45 against 52, 32 55 against 52).  The counts are on the
  // device, so the rule takes all rows; it holds for uneven loads (mx, with half of the rows on one expert of
  // 64 of 2048 x 1408, 4096 rows 40 against 43; 64 of 2 x 1408 x 2048, 2048 rows 55 against 61; 8 of
  // 2 x 14336 x 4096, 256 rows 103 against 122) up to nearly all rows on one (all: 31 against 23, 39
  // against 21, 53 against 35).
  const int64_t few = (int64_t)num_experts * (wq_up ? kFp4DecodeRows / 2 : kFp4DecodeRows);
  return total_rows <= few ? run_fp4_decode(p, stream) : run_fp4_gemm(p, stream);
}
