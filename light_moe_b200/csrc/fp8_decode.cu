// fp8_decode.cu -- grouped product of block-scaled 8-bit operands for few rows per expert (sm_100a).
//
// The same product as fp8_gemm.cu with the operands' roles exchanged: a CTA pair's tile is 256 weight
// rows (128 per CTA, TMEM lane = output feature; with SwiGLU 256 of gate and the same 256 of up) x up to
// 64 rows.  A handful of rows fills a row tile of 256 badly, and what bounds here is the weights' way
// from HBM: a block of 256 x 128 weights is 32 KB a pair, ~700 cycles of all pairs' share of HBM.  The
// row-tile kernel spends ~1000 cycles on a block whatever its rows (its chain of MMA, hand-over, reading
// and adding 128 columns a thread has two buffers to hide in); here an MMA takes 128 cycles, a thread
// reads and adds 32 columns (64 with SwiGLU), and tensor memory holds 8 (4) blocks' sums.
//
// The weights' scale is one number per CTA, matrix and block (128 x 128), the rows' scales are one per
// column: the scales' warp multiplies the two and leaves a block's 64 factors in shared memory, from where
// every thread reads them as broadcasts.
//
// Bound by HBM: 18 rows, 8 experts of 2 x 14336 x 4096, 943 MB in 154 us (6.1 TB/s; tiles of rows 252 us); 128 uneven
// rows, 8 of 4096 x 14336, 473 MB in 93 us, two rounds of 128 tiles on 74 pairs.
//
// Warps: 0 TMA producer, whose copies complete on the leader's stage barrier; 1 MMA issuer (leader
// CTA); 2 scales; 4-11 the epilogue (lane quarter x half of the columns).
#include <cuda_bf16.h>

#include "fp8_format.cuh"
#include "fp8_gemm.h"
#include "pair_gemm.cuh"

namespace lmoe {
namespace {

constexpr int kRowsCta = 128, kTM = 256, kTN = kFp8DecodeRows, kBK = kFp8Block;
constexpr int kEpiWarps = 8, kEpiWarp0 = 4, kThreads = (kEpiWarp0 + kEpiWarps) * 32;
constexpr int kTmemCols = 512;
constexpr int kSlotBlocks = 8, kSlots = 3;
constexpr uint32_t kSite = 0x780u;

template <bool SWIGLU>
struct Cfg {
  static constexpr int kMats = SWIGLU ? 2 : 1;
  static constexpr uint32_t kABytes = kRowsCta * kBK, kBBytes = kTN / 2 * kBK;
  static constexpr uint32_t kStageBytes = kMats * kABytes + kBBytes;
  static constexpr int kStages = SWIGLU ? 5 : 10;
  static constexpr int kAccCols = kMats * kTN, kAcc = kTmemCols / kAccCols;
};

template <class C>
struct ScaleSlot {
  float factor[kSlotBlocks][C::kMats][kTN];   // of the rows times this CTA's weights
};

template <class C>
struct __align__(8) Bars {
  uint64_t full[C::kStages];      // leader: both CTAs' codes landed (one arrival each)
  uint64_t empty[C::kStages];     // the stage's MMAs finished (both CTAs)
  uint64_t acc_full[C::kAcc];     // a block's sums are in tensor memory (both CTAs)
  uint64_t acc_empty[C::kAcc];    // leader: both CTAs' epilogue warps have read them
  uint64_t sc_full[kSlots];       // this CTA: the slot's factors are written
  uint64_t sc_empty[kSlots];      // this CTA: its epilogue warps have read them
  uint64_t mma_done;
  uint32_t tmem_base;
  int abort;
  SegTable seg;
};

template <class C>
constexpr uint32_t smem_bytes() {
  return 1024 + C::kStages * C::kStageBytes + kSlots * sizeof(ScaleSlot<C>) + sizeof(Bars<C>);
}
static_assert(smem_bytes<Cfg<false>>() <= 232448 && smem_bytes<Cfg<true>>() <= 232448, "shared memory budget");
static_assert(Cfg<false>::kStageBytes % 1024 == 0 && Cfg<true>::kStageBytes % 1024 == 0, "swizzle atoms");

struct Args {
  const float* xs;
  int64_t xs_pitch;
  const float* ws;       // [E, NB, KB]; gate
  const float* ws_up;
  const void* offsets;
  int offsets_i64;
  int E, N, KB, NB;
  int64_t R;
  Raster raster;         // of the feature tiles
  void* out;
  int out_dtype;
  uint32_t* err;
};

struct Tile {
  int e, m, n, row0, row_end;
  bool zero;   // rows outside every expert
};
__device__ __forceinline__ Tile tile_at(const SegTable& t, const Args& a, int tile, int& hint) {
  int j = hint;
  while (tile >= t.tile_start[j + 1]) ++j;
  hint = j;
  Tile r;
  const int rows = t.row[j + 1] - t.row[j];
  a.raster.at(tile - t.tile_start[j], (rows + kTN - 1) / kTN, r.m, r.n);
  r.e = j - 1;
  r.zero = j == 0 || j == a.E + 1;
  r.row0 = t.row[j] + r.m * kTN;
  r.row_end = t.row[j + 1];
  return r;
}

// acc += f * r for 32 values, each with its own factor (broadcast from shared memory).
__device__ __forceinline__ void add_scaled(float* acc, const uint32_t (&r)[32], const float* f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 v = reinterpret_cast<const float4*>(f)[i];
    acc[4 * i] = fmaf(__uint_as_float(r[4 * i]), v.x, acc[4 * i]);
    acc[4 * i + 1] = fmaf(__uint_as_float(r[4 * i + 1]), v.y, acc[4 * i + 1]);
    acc[4 * i + 2] = fmaf(__uint_as_float(r[4 * i + 2]), v.z, acc[4 * i + 2]);
    acc[4 * i + 3] = fmaf(__uint_as_float(r[4 * i + 3]), v.w, acc[4 * i + 3]);
  }
}

template <bool SWIGLU>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    fp8_decode_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                      const __grid_constant__ CUtensorMap tm_up, const Args a) {
  using C = Cfg<SWIGLU>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  ScaleSlot<C>* slots = reinterpret_cast<ScaleSlot<C>*>(base + C::kStages * C::kStageBytes);
  Bars<C>* bars = reinterpret_cast<Bars<C>*>(slots + kSlots);
  volatile int* abort_flag = &bars->abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (tid == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&bars->full[s], 2);
      mbar_init(&bars->empty[s], 1);
    }
    for (int s = 0; s < C::kAcc; ++s) {
      mbar_init(&bars->acc_full[s], 1);
      mbar_init(&bars->acc_empty[s], 2 * kEpiWarps);
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&bars->sc_full[s], 1);
      mbar_init(&bars->sc_empty[s], kEpiWarps);
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
      return (bars->seg.row[j + 1] - bars->seg.row[j] + kTN - 1) / kTN * a.raster.nb;
    });
  if (tid == 0 && bars->seg.bad && blockIdx.x == 0) report_error(a.err, kErrBadArg, kSite + 1);
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  const SegTable& seg = bars->seg;
  const int total = seg.tile_start[segs];
  const int KB = a.KB;
  const int first = blockIdx.x >> 1, stride = gridDim.x >> 1;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    const uint32_t full_addr = mapa_u32(&bars->full[0], 0);
    Ring<C::kStages> st;
    int hint = 0;
    bool ok = true;
    for (int tile = first; tile < total && ok; tile += stride) {
      const Tile t = tile_at(seg, a, tile, hint);
      if (t.zero) continue;
      const int wrow = t.n * kTM + (int)rank * kRowsCta, row = t.row0 + (int)rank * (kTN / 2);
      const bool rows = row < t.row_end;   // of this CTA's half of the columns
      for (int kb = 0; kb < KB; ++kb, st.next()) {
        ok = warp_wait(&bars->empty[st.i], st.phase ^ 1u, a.err, abort_flag, kSite + 2);
        if (!ok) break;
        if (elect_one()) {
          uint8_t* dst = base + st.i * C::kStageBytes;
          const uint32_t bar = full_addr + st.i * 8;
          mbar_arrive_expect_tx_cluster(bar, C::kMats * C::kABytes + (rows ? C::kBBytes : 0u));
          tma_load_3d_pair(dst, &tm_w, bar, kb * kBK, wrow, t.e);
          if (SWIGLU) tma_load_3d_pair(dst + C::kABytes, &tm_up, bar, kb * kBK, wrow, t.e);
          if (rows) tma_load_2d_pair(dst + C::kMats * C::kABytes, &tm_x, bar, kb * kBK, row);
        }
      }
    }
    // the copies of a finished tile have landed (its MMAs read them)
    if (!ok) let_copies_land();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (leader) {
      const uint64_t adesc0 = sdesc_k_sw128(smem_u32(base));
      const uint64_t bdesc0 = sdesc_k_sw128(smem_u32(base) + C::kMats * C::kABytes);
      Ring<C::kStages> st;
      Ring<C::kAcc> ac;
      int blocks = 0, hint = 0;   // of all this pair's tiles
      for (int tile = first; tile < total; tile += stride)
        if (!tile_at(seg, a, tile, hint).zero) blocks += KB;
      bool ok = true;
      for (; blocks > 0; --blocks) {
        // the waits start together; what has not come yet is waited for below
        const bool w0 = mbar_test(&bars->acc_empty[ac.i], ac.phase ^ 1u);
        const bool w1 = mbar_test(&bars->full[st.i], st.phase);
        if (!(w0 && w1)) {
          ok = mbar_wait(&bars->acc_empty[ac.i], ac.phase ^ 1u, a.err, abort_flag, kSite + 3);
          if (ok) ok = mbar_wait(&bars->full[st.i], st.phase, a.err, abort_flag, kSite + 4);
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t ad = adesc0 + st.i * (C::kStageBytes >> 4), bd = bdesc0 + st.i * (C::kStageBytes >> 4);
          const uint32_t d = tmem + ac.i * C::kAccCols;
#pragma unroll
          for (int u = 0; u < C::kMats; ++u)
#pragma unroll
            for (int m = 0; m < kBK / 32; ++m)   // 32 bytes of the lines: two descriptor units
              mma_fp8_pair(d + u * kTN, ad + u * (C::kABytes >> 4) + m * 2, bd + m * 2, idesc_fp8(kTN),
                           (uint32_t)(m > 0));
          mma_commit_pair(&bars->acc_full[ac.i]);
          mma_commit_pair(&bars->empty[st.i]);
        }
        __syncwarp();
        st.next();
        ac.next();
      }
      if (elect_one()) mma_commit_leader(&bars->mma_done);
      mbar_wait(&bars->mma_done, 0, a.err, nullptr, kSite + 5);
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ scales
    Ring<kSlots> sl;
    int hint = 0;
    bool ok = true;
    for (int tile = first; tile < total && ok; tile += stride) {
      const Tile t = tile_at(seg, a, tile, hint);
      if (t.zero) continue;
      const int nb = t.n * 2 + (int)rank;   // a CTA's rows are one block of the weights' scales
      const float* w = a.ws + ((int64_t)t.e * a.NB + (nb < a.NB ? nb : a.NB - 1)) * KB;
      const float* wu = SWIGLU ? a.ws_up + (w - a.ws) : w;
      for (int kb = 0; kb < KB; kb += kSlotBlocks, sl.next()) {
        float v[kSlotBlocks][2], g = 0.0f, u = 0.0f;
#pragma unroll
        for (int j = 0; j < kSlotBlocks; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int row = t.row0 + i * 32 + lane;
            v[j][i] = kb + j < KB && row < t.row_end ? __ldg(a.xs + (int64_t)(kb + j) * a.xs_pitch + row) : 0.0f;
          }
        if (lane < kSlotBlocks && kb + lane < KB) {
          g = __ldg(w + kb + lane);
          if (SWIGLU) u = __ldg(wu + kb + lane);
        }
        ok = warp_wait(&bars->sc_empty[sl.i], sl.phase ^ 1u, a.err, abort_flag, kSite + 6);
        if (!ok) break;
#pragma unroll
        for (int j = 0; j < kSlotBlocks; ++j) {
          const float gj = __shfl_sync(0xffffffffu, g, j), uj = __shfl_sync(0xffffffffu, u, j);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            slots[sl.i].factor[j][0][i * 32 + lane] = __fmul_rn(v[j][i], gj);
            if (SWIGLU) slots[sl.i].factor[j][C::kMats - 1][i * 32 + lane] = __fmul_rn(v[j][i], uj);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->sc_full[sl.i]);   // (release: the warp's stores are before it)
      }
    }
  } else if (warp >= kEpiWarp0) {
    // ------------------------------------------------------------------ epilogue
    const int q = warp & 3, half = (warp - kEpiWarp0) >> 2;
    const uint32_t mine = tmem + ((uint32_t)(q * 32) << 16) + half * 32;
    const uint32_t empty_addr = mapa_u32(&bars->acc_empty[0], 0);
    Ring<C::kAcc> ac;
    Ring<kSlots> sl;
    int hint = 0, in_slot = 0;
    bool ok = true;
    for (int tile = first; tile < total; tile += stride) {
      const Tile t = tile_at(seg, a, tile, hint);
      const int row = t.row0 + half * 32;   // the warp's first column
      const int rows = t.row_end - row < 32 ? t.row_end - row : 32;
      const int feature = t.n * kTM + (int)rank * kRowsCta + q * 32 + lane;
      float acc[C::kMats * 32];
#pragma unroll
      for (int i = 0; i < C::kMats * 32; ++i) acc[i] = 0.0f;
      if (!t.zero && ok) {
        for (int left = KB; left > 0; --left) {
          if (in_slot == 0) ok = mbar_wait(&bars->sc_full[sl.i], sl.phase, a.err, abort_flag, kSite + 7);
          ok = ok && mbar_wait(&bars->acc_full[ac.i], ac.phase, a.err, abort_flag, kSite + 8);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          uint32_t r[C::kMats][32];
          if (rows > 0) {   // else there are no rows in this half
            if constexpr (SWIGLU)
              tmem_ld32x2(mine + ac.i * C::kAccCols, mine + ac.i * C::kAccCols + kTN, r[0], r[C::kMats - 1]);
            else
              tmem_ld32(mine + ac.i * C::kAccCols, r[0]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(empty_addr + ac.i * 8);
          ac.next();
          if (rows > 0) {
#pragma unroll
            for (int u = 0; u < C::kMats; ++u)
              add_scaled(acc + u * 32, r[u], &slots[sl.i].factor[in_slot][u][half * 32]);
          }
          if (++in_slot == kSlotBlocks || left == 1) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->sc_empty[sl.i]);
            sl.next();
            in_slot = 0;
          }
        }
      }
      if (!t.zero && !ok) {   // what was not computed is NaN
#pragma unroll
        for (int i = 0; i < C::kMats * 32; ++i) acc[i] = __uint_as_float(0x7fc00000u);
      }
      if (feature >= a.N) continue;
      // a row's 32 features of a warp are neighbours
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        if (j >= rows) break;
        float v = acc[j];
        if (SWIGLU) v = __fdividef(v, 1.0f + __expf(-v)) * acc[(C::kMats - 1) * 32 + j];
        const int64_t at = (int64_t)(row + j) * a.N + feature;
        if (a.out_dtype == LMOE_DTYPE_F32)
          static_cast<float*>(a.out)[at] = v;
        else if (a.out_dtype == LMOE_DTYPE_F16)
          static_cast<__half*>(a.out)[at] = __float2half_rn(v);
        else
          static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
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

template <bool SWIGLU>
int launch(const CUtensorMap& x, const CUtensorMap& w, const CUtensorMap& up, const Args& a, int grid,
           cudaStream_t stream) {
  auto fn = fp8_decode_kernel<SWIGLU>;
  const int st = set_max_dynamic_smem(reinterpret_cast<const void*>(fn), smem_bytes<Cfg<SWIGLU>>());
  if (st != LMOE_OK) return st;
  fn<<<grid, kThreads, smem_bytes<Cfg<SWIGLU>>(), stream>>>(x, w, up, a);
  return cuda_status(cudaGetLastError());
}

}  // namespace

int run_fp8_decode(const Fp8Problem& p, cudaStream_t stream) {
  DeviceInfo dev;
  int st = get_device_info(&dev);
  if (st != LMOE_OK) return st;
  if (dev.cc_major != 10) return LMOE_ERR_DEVICE;
  const bool swiglu = p.wq_up != nullptr;
  const int grid = gemm_grid(dev) < 2 ? 2 : gemm_grid(dev) & ~1;   // whole pairs
  Args a = {};
  a.xs = p.xs;
  a.xs_pitch = p.xs_pitch;
  a.ws = p.ws;
  a.ws_up = p.ws_up;
  a.offsets = p.offsets;
  a.offsets_i64 = p.offsets_i64;
  a.E = p.num_experts;
  a.N = p.N;
  a.KB = (p.K + kBK - 1) / kBK;
  a.NB = (p.N + kFp8Block - 1) / kFp8Block;
  a.R = p.total_rows;
  a.raster = Raster((p.N + kTM - 1) / kTM);
  a.out = p.out;
  a.out_dtype = p.out_dtype;
  a.err = p.err;
  CUtensorMap tx, tw, tu;
  const uint64_t kb = (uint64_t)p.K;
  st = encode_tmap_2d(&tx, p.xq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)p.total_rows, kb, kb, kTN / 2, kBK, true);
  if (st != LMOE_OK) return st;
  const uint64_t dims[3] = {kb, (uint64_t)p.N, (uint64_t)p.num_experts};
  const uint64_t strides[2] = {kb, kb * (uint64_t)p.N};
  const uint32_t box[3] = {(uint32_t)kBK, (uint32_t)kRowsCta, 1};
  st = encode_tmap_3d(&tw, p.wq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, dims, strides, box);
  if (st != LMOE_OK) return st;
  tu = tw;
  if (swiglu) {
    st = encode_tmap_3d(&tu, p.wq_up, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, dims, strides, box);
    if (st != LMOE_OK) return st;
  }
  return swiglu ? launch<true>(tx, tw, tu, a, grid, stream) : launch<false>(tx, tw, tu, a, grid, stream);
}

}  // namespace lmoe
