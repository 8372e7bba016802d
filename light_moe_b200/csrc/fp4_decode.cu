// fp4_decode.cu -- grouped product of microscaled 4-bit operands for few rows per expert (sm_100a).
//
// The same product as fp4_gemm.cu with the operands' roles exchanged: the MMA's M runs over 256
// weight rows of a CTA pair (128 per CTA) and N over up to 64 rows of the batch, so a stage holds
// weights, not padding of the batch to 256 rows, and an MMA takes 32 cycles.  Bound by reading the
// weights (HBM): four stages of 32 KB of codes per SM are in flight (8 experts of 2 x 14336 x 4096,
// a row each: 79 us for 499 MB, 97 % of the measured copy rate).
//
// A CTA's 128 TMEM lanes are 128 features, or (gate / up) 64 gate rows and the same 64 rows of up:
// the up lanes hand their values to the gate lanes through shared memory, and a warp stores 32
// neighbouring features of one row of the batch at a time.
//
// Warps: 0 TMA producer; 1 MMA issuer (leader CTA); 2, 3 scales of the weight rows, 4 scales of the
// batch's 64 rows; 5-8 epilogue.  Barriers, scales and issue order are those of fp4_gemm.cu, with
// four TMEM buffers of a unit's scales (32 columns).
#include <cuda_bf16.h>

#include "fp4_mma.cuh"
#include "host_util.h"

namespace lmoe {
namespace {

constexpr int kRows = kFp4DecodeRows;      // rows of the batch in a tile
constexpr int kStages = 4, kAcc = 2, kSfSlots = 3, kUnits = 4;
constexpr uint32_t kUnitCols = 32;         // 4 words x (4 columns of the weights' scales, 4 of the rows')
constexpr int kSfWarp0 = 2, kSfWarps = 3, kEpiWarp0 = 5, kEpiWarps = 4;
constexpr int kThreads = (kEpiWarp0 + kEpiWarps) * 32;
constexpr uint32_t kABlock = 128 * 128, kBBlock = (kRows / 2) * 128;
constexpr uint32_t kABytes = 2 * kABlock, kBBytes = 2 * kBBlock, kStageBytes = kABytes + kBBytes;
constexpr uint32_t kSfABytes = 8 * 512, kSfSlotBytes = 2 * kSfABytes;
constexpr uint32_t kXchgBytes = 2 * 64 * (kRows + 1) * 4;
constexpr uint32_t kSite = 0x800u;
constexpr int kTmemCols = 256;
static_assert(kAcc * kRows + kUnits * kUnitCols <= kTmemCols, "tensor memory budget");

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
constexpr uint32_t kSmem = 1024 + kStages * kStageBytes + kSfSlots * kSfSlotBytes + kXchgBytes + sizeof(Bars);
static_assert(kSmem <= 232448, "shared memory budget");

__device__ __forceinline__ void store_value(void* out, int64_t i, float v, int dtype) {
  if (dtype == LMOE_DTYPE_F32)
    static_cast<float*>(out)[i] = v;
  else
    static_cast<uint16_t*>(out)[i] = (uint16_t)(pack16(v, 0.0f, dtype == LMOE_DTYPE_F16) & 0xffffu);
}

template <int FORMAT, bool SWIGLU>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    fp4_decode_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                      const __grid_constant__ CUtensorMap tm_up, const Fp4Args a) {
  using C = Fp4Units<FORMAT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sf_base = base + kStages * kStageBytes;
  float* xchg = reinterpret_cast<float*>(sf_base + kSfSlots * kSfSlotBytes);   // [64][kRows + 1]
  Bars* bars = reinterpret_cast<Bars*>(reinterpret_cast<uint8_t*>(xchg) + kXchgBytes);
  volatile int* abort_flag = &bars->abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  constexpr int kFeat = SWIGLU ? 64 : 128;   // features of a CTA's tile

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
      mbar_init(&bars->acc_empty[s], 2 * kEpiWarps);
    }
    mbar_init(&bars->mma_done, 1);
    bars->abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(&bars->tmem_base, kTmemCols);
    tmem_relinquish_pair();
  }
  load_segments(&bars->seg, a.offsets, a.offsets_i64, a.E, a.R, tid, kThreads);
  const int segs = a.E + 2;
  if (warp == 0)
    scan_tiles(&bars->seg, segs, lane, [&](int j) {
      return (bars->seg.row[j + 1] - bars->seg.row[j] + kRows - 1) / kRows * a.raster.nb;
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
      const Fp4Tile t = fp4_tile_at<kRows>(seg, a, tile, hint);
      if (t.zero) continue;
      const int r0 = t.row0 + (int)rank * (kRows / 2);   // this CTA's half of the batch's rows
      const bool rows = r0 < t.row_end;
      const int f0 = t.n * 2 * kFeat + (int)rank * kFeat;
      for (int ks = 0; ks < a.KS; ++ks, st.next()) {
        ok = warp_wait(&bars->empty[st.i], st.phase ^ 1u, a.err, abort_flag, kSite + 2);
        if (!ok) break;
        if (elect_one()) {
          uint8_t* dst = base + st.i * kStageBytes;
          const uint32_t bar = full_addr + st.i * 8;
          const int blocks = a.K - ks * kFp4Stage > kFp4Block ? 2 : 1;
          mbar_arrive_expect_tx_cluster(bar, (uint32_t)blocks * (kABlock + (rows ? kBBlock : 0u)));
          for (int h = 0; h < blocks; ++h) {
            const int x = ks * (kFp4Stage / 2) + h * 128;
            tma_load_3d_pair(dst + h * kABlock, &tm_w, bar, x, f0, t.e);
            tma_load_3d_pair(dst + h * kABlock + kABlock / 2, SWIGLU ? &tm_up : &tm_w, bar, x, SWIGLU ? f0 : f0 + 64,
                             t.e);
            if (rows) tma_load_2d_pair(dst + kABytes + h * kBBlock, &tm_x, bar, x, r0);
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
        const Fp4Tile t = fp4_tile_at<kRows>(seg, a, tile, hint);
        if (t.zero) continue;
        ok = warp_wait(&bars->acc_empty[ac.i], ac.phase ^ 1u, a.err, abort_flag, kSite + 4);
        const uint32_t d = tmem + ac.i * kRows;
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
              const uint32_t sfa = tmem + kAcc * kRows + un.i * kUnitCols, sfb = sfa + 16;
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                const int q = 4 * j + w;   // word of the step
                copy_scales_pair(sfa + w * 4, sa + q * 32);
                copy_scales_pair(sfb + w * 4, sb + q * 32);
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
                    mma_fp4_pair<FORMAT>(d, am, bm, idesc_fp4(true, (m & 1) * 2, kRows), sfa + (m >> 1) * 4,
                                         sfb + (m >> 1) * 4, accum | (uint32_t)(m > 0));
                  else
                    mma_fp4_pair<FORMAT>(d, am, bm, idesc_fp4(false, 0, kRows), sfa + m * 4, sfb + m * 4,
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
    const int part = warp - kSfWarp0;   // 0, 1: the first and last 64 weight rows (gate and up); 2: the batch's
    int hint = 0;
    write_scales<FORMAT, kSfSlots>(
        first, total, stride, a.K, sf_base + lane * 16 + (part < 2 ? part * 8u : kSfABytes), 512u, kSfSlotBytes,
        bars->sf_empty, mapa_u32(&bars->sf_full[0], 0), a.err, abort_flag, kSite + 8, lane,
        [&](int tile, const uint8_t* (&p)[2]) {
          const Fp4Tile t = fp4_tile_at<kRows>(seg, a, tile, hint);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = lane + 32 * i;
            p[i] = nullptr;
            if (part == 2) {
              if (t.row0 + r < t.row_end) p[i] = a.xs + (int64_t)(t.row0 + r) * a.xs_pitch;
            } else if (!t.zero) {
              const int f = t.n * 2 * kFeat + (int)rank * kFeat + (SWIGLU ? r : part * 64 + r);
              if (f < a.N) p[i] = (SWIGLU && part == 1 ? a.ws_up : a.ws) + ((int64_t)t.e * a.N + f) * a.ws_pitch;
            }
          }
          return !t.zero;
        });
  } else {
    // ------------------------------------------------------------------ epilogue
    const int q = warp & 3;
    const uint32_t lane_base = (uint32_t)(q * 32) << 16;
    const uint32_t empty_addr = mapa_u32(&bars->acc_empty[0], 0);
    const bool up = SWIGLU && q >= 2;
    const int l = SWIGLU ? (q & 1) * 32 + lane : q * 32 + lane;   // feature within the CTA's tile
    uint32_t turn = 0;
    Ring<kAcc> ac;
    int hint = 0;
    bool ok = true;
    for (int tile = first; tile < total; tile += stride) {
      const Fp4Tile t = fp4_tile_at<kRows>(seg, a, tile, hint);
      const int rows = t.row_end - t.row0 < kRows ? t.row_end - t.row0 : kRows;
      const int f = t.n * 2 * kFeat + (int)rank * kFeat + l;
      uint32_t u[32], v[32];
      float al = 1.0f;
      if (!t.zero) {
        // all four warps leave together: the exchange below has barriers among them
        ok = mbar_wait(&bars->acc_full[ac.i], ac.phase, a.err, abort_flag, kSite + 10);
        if (named_bar_any(1, kEpiWarps * 32, !ok)) break;
        tc_fence_after();
        const uint32_t col = tmem + lane_base + ac.i * kRows;
        tmem_ld32x2(col, col + 32, u, v);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(empty_addr + ac.i * 8);
        ac.next();
        const float* ap = up ? a.alpha_up : a.alpha;
        if (ap) al = __ldg(ap + t.e);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) u[i] = v[i] = 0u;
      }
      // eight rows of the batch at a time, as many as the tile has; two exchange buffers in turn, so
      // that one barrier a tile orders writes, reads and the writes of the tile after next
      float* xb = xchg + (turn & 1u) * (64 * (kRows + 1)) + l * (kRows + 1);
      ++turn;
      if (SWIGLU) {
        if (up) {
#pragma unroll
          for (int i0 = 0; i0 < kRows; i0 += 8) {
            if (i0 < rows) {
#pragma unroll
              for (int i = i0; i < i0 + 8; ++i) xb[i] = __fmul_rn(__uint_as_float(i < 32 ? u[i & 31] : v[i & 31]), al);
            }
          }
        }
        named_bar_sync(2, kEpiWarps * 32);
      }
      if (!up && f < a.N) {
        const int64_t at = (int64_t)t.row0 * a.N + f;
#pragma unroll
        for (int i0 = 0; i0 < kRows; i0 += 8) {
          if (i0 < rows) {
#pragma unroll
            for (int i = i0; i < i0 + 8; ++i) {
              float x = __fmul_rn(__uint_as_float(i < 32 ? u[i & 31] : v[i & 31]), al);
              if (SWIGLU) x = silu(x) * xb[i];
              if (i < rows) store_value(a.out, at + (int64_t)i * a.N, x, a.out_dtype);
            }
          }
        }
      }
    }
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
int launch(const CUtensorMap& x, const CUtensorMap& w, const CUtensorMap& up, const Fp4Args& a, int grid,
           cudaStream_t stream) {
  auto fn = fp4_decode_kernel<FORMAT, SWIGLU>;
  const int st = set_max_dynamic_smem(reinterpret_cast<const void*>(fn), kSmem);
  if (st != LMOE_OK) return st;
  fn<<<grid, kThreads, kSmem, stream>>>(x, w, up, a);
  return cuda_status(cudaGetLastError());
}

}  // namespace

int run_fp4_decode(const Fp4Problem& p, cudaStream_t stream) {
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
  const int features = swiglu ? 128 : 256;
  a.raster = Raster((p.N + features - 1) / features);
  a.KS = (p.K + kFp4Stage - 1) / kFp4Stage;
  a.alpha = p.alpha;
  a.alpha_up = p.alpha_up;
  a.out = p.out;
  a.out_dtype = p.out_dtype;
  a.err = p.err;
  CUtensorMap tx, tw, tu;
  const uint64_t kb = (uint64_t)p.K / 2;
  st = encode_tmap_2d(&tx, p.xq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)p.total_rows, kb, kb, kRows / 2, 128, true);
  if (st != LMOE_OK) return st;
  const uint64_t dims[3] = {kb, (uint64_t)p.N, (uint64_t)p.num_experts};
  const uint64_t strides[2] = {kb, kb * (uint64_t)p.N};
  const uint32_t box[3] = {128, 64, 1};
  st = encode_tmap_3d(&tw, p.wq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, dims, strides, box);
  if (st != LMOE_OK) return st;
  tu = tw;
  if (swiglu) {
    st = encode_tmap_3d(&tu, p.wq_up, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, dims, strides, box);
    if (st != LMOE_OK) return st;
  }
  const int grid = gemm_grid(dev) < 2 ? 2 : gemm_grid(dev) & ~1;   // whole pairs
  if (p.format == LMOE_FP4_MX)
    return swiglu ? launch<LMOE_FP4_MX, true>(tx, tw, tu, a, grid, stream)
                  : launch<LMOE_FP4_MX, false>(tx, tw, tu, a, grid, stream);
  return swiglu ? launch<LMOE_FP4_NV, true>(tx, tw, tu, a, grid, stream)
                : launch<LMOE_FP4_NV, false>(tx, tw, tu, a, grid, stream);
}

}  // namespace lmoe
