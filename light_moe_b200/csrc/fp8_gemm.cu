// fp8_gemm.cu -- grouped product of block-scaled 8-bit operands on CTA pairs (sm_100a).
//
//   y[r, n] = sum_b sx[r, b] * sw[e, n / 128, b] * sum_{k in block b} x[r, k] * w[e, n, k]
//   y[r, f] = silu(gate[r, f]) * up[r, f]                with a gate and an up matrix
//
// for the rows r of expert e: E4M3 codes, fp32 scales of 128 columns of a row (x) or of 128 x 128
// values (w, fp8_format.cuh).  The scales are any fp32 numbers, so the block-scaled MMA kinds (power
// of two scales) do not apply: the tensor core sums one block of 128 columns at a time in tensor
// memory (exact products, fp32 sums), and the epilogue's warps add each block's sums times
// sx * sw to fp32 accumulators in registers.  So no sum of more than 128 products is left to the
// tensor core, whose additions truncate.
//
// Tile: 256 rows (128 per CTA, TMEM lane = row) x 256 or 128 weight rows (half of them per CTA in
// shared memory).  A block of 256 x 256 x 128 takes the pair's tensor cores 512 cycles.  Meanwhile 8 warps a CTA,
// of 32 rows x 128 columns each, read the block before it from the other half of tensor memory and add it, and a
// half of the columns goes back to its issuer as soon as its four warps have read it.  128 accumulators a thread:
// the epilogue's two warpgroups take the registers that the other warps give up.
//
// What bounds it is the chain of a warp, not the tensor core (half of the cycles), and not the multiply-adds (256 cycles
// of an SM a block): it waits for the half, reads 4 x 32 columns, one load after another since two in flight do not fit
// the registers, so that each load's latency shows, and issues 64 paired multiply-adds.  A block takes ~1000 cycles in
// all (3.19 M cycles for a pair's 97 tiles of 32 blocks).  16384 rows through 8 experts of 2 x 14336 x 4096: 1.9 ms in
// single calls with pauses, 2.0 PFLOP/s, 0.6 of twice the measured bf16 rate; 2.05 ms in 100 calls without, and 2.35 ms
// in a run of seconds, when the power limit has lowered the clock.
//
// The lane being the row, a thread holds a row's gate and up values of the same features, and the
// SwiGLU needs no exchange: the leader's half of the columns is gate rows and the follower's the
// same rows of up.
//
// Warps: 0 TMA producer, whose copies complete on the leader's stage barrier; 1 and 3 MMA issuers
// (leader CTA), one for each half of the columns, so that neither half waits for the other's readers;
// 2 scales (both CTAs), which brings eight blocks' scales at a time into a ring in shared memory,
// coalesced because rows' scales are stored block after block; 4-11 the epilogue.
#include <cuda_bf16.h>

#include "fp8_format.cuh"
#include "fp8_gemm.h"
#include "pair_gemm.cuh"

namespace lmoe {
namespace {

constexpr int kRowsCta = 128, kTM = 256, kBK = kFp8Block;
constexpr int kEpiWarps = 8, kEpiWarp0 = 4, kThreads = (kEpiWarp0 + kEpiWarps) * 32;
constexpr int kTmemCols = 512;
constexpr int kSlotBlocks = 8, kSlots = 3;   // a slot of the scales' ring holds eight blocks
constexpr uint32_t kSite = 0x700u;
// Registers: 384 threads x 168 at launch = 128 x 72 + 256 x 216.
constexpr int kRegsLaunch = 168, kRegsOther = 72, kRegsEpi = 216;
static_assert(128 * kRegsOther + 256 * kRegsEpi <= kThreads * kRegsLaunch, "register split");

template <int TN, bool SWIGLU>
struct Cfg {
  static constexpr int kHalf = TN / 2;                  // columns a CTA loads
  static constexpr int kCols = TN / 2;                  // of an MMA, and of an epilogue thread
  static constexpr int kAcc = kTmemCols / TN;           // blocks' sums in tensor memory
  static constexpr int kOutCols = SWIGLU ? kCols / 2 : kCols;       // of a warp's output
  static constexpr uint32_t kStoreBytes = kOutCols / 32 * 2048;    // a warp's tile on its way out: blocks of 32 rows x 64 bytes
  static constexpr uint32_t kABytes = kRowsCta * kBK, kBBytes = kHalf * kBK, kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = TN == 256 ? (SWIGLU ? 5 : 4) : 6;
};

struct ScaleSlot {
  float row[kSlotBlocks][kRowsCta];
  float col[kSlotBlocks][2];   // of the tile's two column blocks, or of gate and up
};

template <class C>
struct __align__(8) Bars {
  uint64_t full[C::kStages];        // leader: both CTAs' codes landed (one arrival each)
  uint64_t empty[C::kStages];       // both halves' MMAs of the stage finished (both CTAs)
  uint64_t acc_full[2][C::kAcc];    // half of a block's sums is in tensor memory (both CTAs)
  uint64_t acc_empty[2][C::kAcc];   // leader: both CTAs' epilogue warps of the half have read it
  uint64_t sc_full[kSlots];         // this CTA: the slot's scales are written
  uint64_t sc_empty[kSlots];        // this CTA: its epilogue warps have read them
  uint64_t mma_done;
  uint32_t tmem_base;
  int abort;
  SegTable seg;
};

template <class C>
constexpr uint32_t smem_bytes() {
  return 1024 + C::kStages * C::kStageBytes + kEpiWarps * C::kStoreBytes + kSlots * sizeof(ScaleSlot) + sizeof(Bars<C>);
}
static_assert(smem_bytes<Cfg<256, false>>() <= 232448 && smem_bytes<Cfg<256, true>>() <= 232448 &&
                  smem_bytes<Cfg<128, false>>() <= 232448 && smem_bytes<Cfg<128, true>>() <= 232448,
              "shared memory budget");
static_assert(sizeof(ScaleSlot) % 16 == 0, "alignment of what follows");

struct Fp8Args {
  const float* xs;
  int64_t xs_pitch;
  const float* ws;       // [E, NB, KB]; gate
  const float* ws_up;
  const void* offsets;
  int offsets_i64;
  int E, N, KB, NB;
  int64_t R;
  Raster raster;         // of the column tiles
  void* out;
  int out_dtype;
  int store;             // StoreMode
  uint32_t* err;
};

struct Fp8Tile {
  int e, m, n, row0, row_end;
  bool zero;   // rows outside every expert
};
__device__ __forceinline__ Fp8Tile fp8_tile_at(const SegTable& t, const Fp8Args& a, int tile, int& hint) {
  int j = hint;
  while (tile >= t.tile_start[j + 1]) ++j;
  hint = j;
  Fp8Tile r;
  const int rows = t.row[j + 1] - t.row[j];
  a.raster.at(tile - t.tile_start[j], (rows + kTM - 1) / kTM, r.m, r.n);
  r.e = j - 1;
  r.zero = j == 0 || j == a.E + 1;
  r.row0 = t.row[j] + r.m * kTM;
  r.row_end = t.row[j + 1];
  return r;
}

// 32 columns of the thread's lane; the registers hold them after tmem_arrived.
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// Completes the thread's loads; the operands keep uses of the registers behind it.
__device__ __forceinline__ void tmem_arrived(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// acc[i] += f * r[i] for 32 values, two to an instruction.
__device__ __forceinline__ void add_scaled(float* acc, const uint32_t (&r)[32], float f) {
  uint64_t f2;
  asm("mov.b64 %0, {%1, %1};" : "=l"(f2) : "f"(f));
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    uint64_t p, c;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "r"(r[2 * i]), "r"(r[2 * i + 1]));
    asm("mov.b64 %0, {%1, %2};" : "=l"(c) : "f"(acc[2 * i]), "f"(acc[2 * i + 1]));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(p), "l"(f2));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(acc[2 * i]), "=f"(acc[2 * i + 1]) : "l"(c));
  }
}

__device__ __forceinline__ float silu(float g) { return __fdividef(g, 1.0f + __expf(-g)); }

template <int TN, bool SWIGLU>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_x32,
                    const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_up,
                    const __grid_constant__ CUtensorMap tm_out, const Fp8Args a) {
  using C = Cfg<TN, SWIGLU>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* store_stage = base + C::kStages * C::kStageBytes;
  ScaleSlot* slots = reinterpret_cast<ScaleSlot*>(store_stage + kEpiWarps * C::kStoreBytes);
  Bars<C>* bars = reinterpret_cast<Bars<C>*>(slots + kSlots);
  volatile int* abort_flag = &bars->abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (tid == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&bars->full[s], 2);
      mbar_init(&bars->empty[s], 2);
    }
    for (int h = 0; h < 2; ++h)
      for (int s = 0; s < C::kAcc; ++s) {
        mbar_init(&bars->acc_full[h][s], 1);
        mbar_init(&bars->acc_empty[h][s], kEpiWarps);
      }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&bars->sc_full[s], 1);
      mbar_init(&bars->sc_empty[s], kEpiWarps);
    }
    mbar_init(&bars->mma_done, 2);   // both issuers
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
  const int KB = a.KB;
  const int first = blockIdx.x >> 1, stride = gridDim.x >> 1;

  if (warp < kEpiWarp0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == 0) {
      // ---------------------------------------------------------------- TMA producer
      const uint32_t full_addr = mapa_u32(&bars->full[0], 0);
      const CUtensorMap* wmap = SWIGLU && !leader ? &tm_up : &tm_w;
      Ring<C::kStages> st;
      int hint = 0;
      bool ok = true;
      for (int tile = first; tile < total && ok; tile += stride) {
        const Fp8Tile t = fp8_tile_at(seg, a, tile, hint);
        if (t.zero) continue;
        const int r0 = t.row0 + (int)rank * kRowsCta;
        int rows = t.row_end - r0;
        rows = rows < 0 ? 0 : (rows > kRowsCta ? kRowsCta : rows);
        const int boxes = (rows + 31) >> 5;   // only the boxes that hold this tile's rows
        const int wrow = SWIGLU ? t.n * C::kHalf : t.n * TN + (int)rank * C::kHalf;
        for (int kb = 0; kb < KB; ++kb, st.next()) {
          ok = warp_wait(&bars->empty[st.i], st.phase ^ 1u, a.err, abort_flag, kSite + 2);
          if (!ok) break;
          if (elect_one()) {
            uint8_t* dst = base + st.i * C::kStageBytes;
            const uint32_t bar = full_addr + st.i * 8;
            mbar_arrive_expect_tx_cluster(bar, (uint32_t)boxes * 4096u + C::kBBytes);
            if (boxes == 4) {
              tma_load_2d_pair(dst, &tm_x, bar, kb * kBK, r0);
            } else {
              for (int b = 0; b < boxes; ++b) tma_load_2d_pair(dst + b * 4096, &tm_x32, bar, kb * kBK, r0 + b * 32);
            }
            tma_load_3d_pair(dst + C::kABytes, wmap, bar, kb * kBK, wrow, t.e);
          }
        }
      }
      // the copies of a finished tile have landed (its MMAs read them)
      if (!ok) let_copies_land();
    } else if (warp == 1 || warp == 3) {
      // ---------------------------------------------------------------- MMA issuers, one for each half of the columns
      if (leader) {
        const int h = warp >> 1;
        const uint64_t adesc0 = sdesc_k_sw128(smem_u32(base));
        const uint64_t bdesc0 = sdesc_k_sw128(smem_u32(base) + C::kABytes + h * (C::kHalf / 2 * kBK));
        Ring<C::kStages> st;
        Ring<C::kAcc> ac;
        int blocks = 0, hint = 0;   // of all this pair's tiles
        for (int tile = first; tile < total; tile += stride)
          if (!fp8_tile_at(seg, a, tile, hint).zero) blocks += KB;
        bool ok = true;
        for (; blocks > 0; --blocks) {
          // the waits start together; what has not come yet is waited for below
          const bool w0 = mbar_test(&bars->acc_empty[h][ac.i], ac.phase ^ 1u);
          const bool w1 = mbar_test(&bars->full[st.i], st.phase);
          if (!(w0 && w1)) {
            ok = mbar_wait(&bars->acc_empty[h][ac.i], ac.phase ^ 1u, a.err, abort_flag, kSite + 3);
            if (ok) ok = mbar_wait(&bars->full[st.i], st.phase, a.err, abort_flag, kSite + 4);
          }
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t ad = adesc0 + st.i * (C::kStageBytes >> 4), bd = bdesc0 + st.i * (C::kStageBytes >> 4);
            const uint32_t d = tmem + (ac.i * 2 + h) * C::kCols;
#pragma unroll
            for (int m = 0; m < kBK / 32; ++m)   // 32 bytes of the lines: two descriptor units
              mma_fp8_pair(d, ad + m * 2, bd + m * 2, idesc_fp8(C::kCols), (uint32_t)(m > 0));
            mma_commit_pair(&bars->acc_full[h][ac.i]);
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
      // ---------------------------------------------------------------- scales
      Ring<kSlots> sl;
      int hint = 0;
      bool ok = true;
      for (int tile = first; tile < total && ok; tile += stride) {
        const Fp8Tile t = fp8_tile_at(seg, a, tile, hint);
        if (t.zero) continue;
        const int r0 = t.row0 + (int)rank * kRowsCta;
        // lanes 0-7: the slot's scales of the first columns (gate), 8-15 of the second (up)
        const int nb0 = SWIGLU ? t.n * C::kHalf / kFp8Block : t.n * TN / kFp8Block;
        const int nb1 = SWIGLU || TN == 128 ? nb0 : nb0 + 1;
        const int nb = (lane & 8) ? (nb1 < a.NB ? nb1 : a.NB - 1) : nb0;
        const float* ws = (SWIGLU && (lane & 8) ? a.ws_up : a.ws) + ((int64_t)t.e * a.NB + nb) * KB + (lane & 7);
        for (int kb = 0; kb < KB; kb += kSlotBlocks, sl.next()) {
          ok = warp_wait(&bars->sc_empty[sl.i], sl.phase ^ 1u, a.err, abort_flag, kSite + 6);
          if (!ok) break;
          ScaleSlot* s = slots + sl.i;
          if (lane < 16) s->col[lane & 7][lane >> 3] = kb + (lane & 7) < KB ? __ldg(ws + kb) : 0.0f;
#pragma unroll
          for (int j0 = 0; j0 < kSlotBlocks; j0 += 2) {
            float v[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int row = r0 + i * 32 + lane;
                v[j][i] = kb + j0 + j < KB && row < t.row_end ? __ldg(a.xs + (int64_t)(kb + j0 + j) * a.xs_pitch + row) : 0.0f;
              }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int i = 0; i < 4; ++i) s->row[j0 + j][i * 32 + lane] = v[j][i];
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->sc_full[sl.i]);   // (release: the warp's stores are before it)
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpi));
    const int q = warp & 3, half = (warp - kEpiWarp0) >> 2;
    const uint32_t lane_base = (uint32_t)(q * 32) << 16;
    const uint32_t empty_addr = mapa_u32(&bars->acc_empty[half][0], 0);
    const int64_t pitch = (int64_t)a.N * (a.out_dtype == LMOE_DTYPE_F32 ? 4 : 2);
    uint8_t* stage = store_stage + (warp - kEpiWarp0) * C::kStoreBytes;
    constexpr int kChunks = C::kCols / 32, kPart = kChunks / 2;
    // first column of chunk c in the tile: the half's rows of the leader's, then of the follower's operand
    auto column = [&](int c) { return c / kPart * C::kHalf + half * (C::kHalf / 2) + c % kPart * 32; };
    Ring<C::kAcc> ac;
    Ring<kSlots> sl;
    int hint = 0, in_slot = 0;
    float f0 = 0.0f, f1 = 0.0f;
    bool ok = true;
    // A lane whose wait ran out still takes every step of its tile with the others, since the loads of tensor memory
    // need the whole warp, but waits no more; lane 0 then gives nothing back.  The warp agrees at the tile's end (with a
    // vote every block the prompt's product took 0.7 % longer).
    // Waits for the next block's sums and reads its factors.
    auto next_block = [&]() {
      if (in_slot == 0) ok = ok && mbar_wait(&bars->sc_full[sl.i], sl.phase, a.err, abort_flag, kSite + 7);
      const ScaleSlot* s = slots + sl.i;
      const float sx = s->row[in_slot][q * 32 + lane];
      const float2 w = *reinterpret_cast<const float2*>(s->col[in_slot]);
      f0 = __fmul_rn(sx, w.x);
      f1 = __fmul_rn(sx, w.y);
      ok = ok && mbar_wait(&bars->acc_full[half][ac.i], ac.phase, a.err, abort_flag, kSite + 8);
      __syncwarp();
      tc_fence_after();
    };
    // Gives the block's sums back, and its factors' slot.
    auto pass_block = [&](bool last) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0 && ok) mbar_arrive_cluster(empty_addr + ac.i * 8);
      ac.next();
      if (++in_slot == kSlotBlocks || last) {
        if (lane == 0 && ok) mbar_arrive(&bars->sc_empty[sl.i]);
        sl.next();
        in_slot = 0;
      }
    };
    for (int tile = first; tile < total; tile += stride) {
      const Fp8Tile t = fp8_tile_at(seg, a, tile, hint);
      const int row = t.row0 + (int)rank * kRowsCta + q * 32;   // the warp's first
      const int rows = t.row_end - row < 32 ? t.row_end - row : 32;
      float acc[C::kCols];
#pragma unroll
      for (int i = 0; i < C::kCols; ++i) acc[i] = 0.0f;
      if (!t.zero && ok) {
        next_block();
        if (rows <= 0) {   // the segment ends before this warp's rows
          for (int left = KB; left > 0; --left) {
            pass_block(left == 1);
            if (left > 1) next_block();
          }
        } else {
          // 32 columns at a time
          const uint32_t lanes = tmem + lane_base + half * C::kCols;
          for (int left = KB; left > 0; --left) {
            const uint32_t col = lanes + ac.i * TN;
            const float g0 = f0, g1 = f1;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
              uint32_t r[32];
              tmem_ld32_async(col + c * 32, r);
              tmem_arrived(r);
              if (c == kChunks - 1) pass_block(left == 1);
              add_scaled(acc + c * 32, r, c < kPart ? g0 : g1);
            }
            if (left > 1) next_block();
          }
        }
        ok = __all_sync(0xffffffffu, ok);
      }
      if (rows <= 0) continue;
      if (!t.zero && !ok) {   // what was not computed is NaN
#pragma unroll
        for (int i = 0; i < C::kCols; ++i) acc[i] = __uint_as_float(0x7fc00000u);
      }
      constexpr int kOut = SWIGLU ? kPart : kChunks;
      if (SWIGLU) {
#pragma unroll
        for (int i = 0; i < C::kCols / 2; ++i) acc[i] = silu(acc[i]) * acc[C::kCols / 2 + i];
      }
      uint8_t* out = static_cast<uint8_t*>(a.out) + (int64_t)row * pitch;
      const bool whole = rows == 32 && a.store != kStoreStaged;   // blocks leave by TMA
      const int c0 = t.n * (SWIGLU ? C::kHalf : TN);
      if (elect_one()) bulk_wait_read();   // of the last tile's stores
      __syncwarp();
      if (!whole) {
#pragma unroll
        for (int b = 0; b < kOut; ++b)
          store_rows<32, C::kStoreBytes>(out, pitch, rows, c0 + column(b), a.N, reinterpret_cast<const float(&)[32]>(acc[b * 32]),
                                         a.out_dtype, a.store, stage, lane);
      } else if (a.out_dtype != LMOE_DTYPE_F32) {
        // all blocks into shared memory, then out together
#pragma unroll
        for (int b = 0; b < kOut; ++b) stage_block<64>(acc + b * 32, a.out_dtype, stage + b * 2048, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (elect_one()) {
#pragma unroll
          for (int b = 0; b < kOut; ++b)
            if (c0 + column(b) < a.N) tma_store_3d(&tm_out, stage + b * 2048, c0 + column(b), row, 0);
          bulk_commit();
        }
        __syncwarp();
      } else {
#pragma unroll
        for (int b = 0; b < 2 * kOut; ++b) {
          const int c = c0 + column(b / 2) + b % 2 * 16;
          if (c < a.N) store_block<64>(&tm_out, acc + b * 16, a.out_dtype, stage, lane, c, row, 0);
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

template <int TN, bool SWIGLU>
int launch(const CUtensorMap& x, const CUtensorMap& x32, const CUtensorMap& w, const CUtensorMap& up,
           const CUtensorMap& out, const Fp8Args& a, int grid, cudaStream_t stream) {
  auto fn = fp8_gemm_kernel<TN, SWIGLU>;
  const int st = set_max_dynamic_smem(reinterpret_cast<const void*>(fn), smem_bytes<Cfg<TN, SWIGLU>>());
  if (st != LMOE_OK) return st;
  fn<<<grid, kThreads, smem_bytes<Cfg<TN, SWIGLU>>(), stream>>>(x, x32, w, up, out, a);
  return cuda_status(cudaGetLastError());
}

}  // namespace

int run_fp8_gemm(const Fp8Problem& p, cudaStream_t stream) {
  DeviceInfo dev;
  int st = get_device_info(&dev);
  if (st != LMOE_OK) return st;
  if (dev.cc_major != 10) return LMOE_ERR_DEVICE;
  const bool swiglu = p.wq_up != nullptr;
  const int grid = gemm_grid(dev) < 2 ? 2 : gemm_grid(dev) & ~1;   // whole pairs
  const int widths[2] = {256, 128};
  const int mats = swiglu ? 2 : 1;
  // A block of a narrow tile takes about four fifths of a wide one's time (8 experts of 2 x 14336 x 4096, 18 rows: 322 us
  // with narrow tiles, 252 with wide ones; 16384 rows: 3090 against 2290), so they pay only where they save a round.
  const int tn = pick_width(widths, grid / 2, 200, 0, [&](int w) {
    return even_row_tiles(p.total_rows, p.num_experts, kTM) * (((int64_t)p.N * mats + w - 1) / w);
  });
  Fp8Args a = {};
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
  a.raster = Raster((int)(((int64_t)p.N * mats + tn - 1) / tn));
  a.out = p.out;
  a.out_dtype = p.out_dtype;
  a.store = store_mode(p.out, p.N, p.out_dtype);
  a.err = p.err;
  CUtensorMap tx, tx32, tw, tu, to = {};
  if (a.store != kStoreStaged) {
    st = encode_store_map(&to, p.out, p.out_dtype, (uint64_t)p.N, (uint64_t)p.total_rows, 1, 64);
    if (st != LMOE_OK) return st;
  }
  const uint64_t kb = (uint64_t)p.K;
  st = encode_tmap_2d(&tx, p.xq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)p.total_rows, kb, kb, kRowsCta, kBK, true);
  if (st != LMOE_OK) return st;
  st = encode_tmap_2d(&tx32, p.xq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)p.total_rows, kb, kb, 32, kBK, true);
  if (st != LMOE_OK) return st;
  const uint64_t dims[3] = {kb, (uint64_t)p.N, (uint64_t)p.num_experts};
  const uint64_t strides[2] = {kb, kb * (uint64_t)p.N};
  const uint32_t box[3] = {(uint32_t)kBK, (uint32_t)tn / 2, 1};
  st = encode_tmap_3d(&tw, p.wq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, dims, strides, box);
  if (st != LMOE_OK) return st;
  tu = tw;
  if (swiglu) {
    st = encode_tmap_3d(&tu, p.wq_up, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, dims, strides, box);
    if (st != LMOE_OK) return st;
  }
  if (tn == 256)
    return swiglu ? launch<256, true>(tx, tx32, tw, tu, to, a, grid, stream)
                  : launch<256, false>(tx, tx32, tw, tu, to, a, grid, stream);
  return swiglu ? launch<128, true>(tx, tx32, tw, tu, to, a, grid, stream)
                : launch<128, false>(tx, tx32, tw, tu, to, a, grid, stream);
}

}  // namespace lmoe

using namespace lmoe;

extern "C" int lmoe_fp8_grouped_gemm(const uint8_t* xq, const float* xs, int64_t xs_pitch, int64_t total_rows, int K,
                                     const uint8_t* wq, const float* ws, const uint8_t* wq_up, const float* ws_up,
                                     int N, const void* expert_offsets, int offsets_are_int64, int num_experts,
                                     int out_dtype, void* output, uint32_t* error, lmoe_stream_t stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  LMOE_ARG_CHECK(out_dtype == LMOE_DTYPE_BF16 || out_dtype == LMOE_DTYPE_F16 || out_dtype == LMOE_DTYPE_F32);
  LMOE_ARG_CHECK(total_rows >= 0 && N > 0 && K > 0 && K % 16 == 0);
  // indexes of whole tiles and stages stay within 32 bits
  LMOE_ARG_CHECK(total_rows <= kMaxGemmSize && N <= kMaxGemmSize / 2 && K <= kMaxGemmSize);
  LMOE_ARG_CHECK(num_experts >= 1);
  if (num_experts > kMaxGemmExperts) return LMOE_ERR_UNSUPPORTED;
  LMOE_ARG_CHECK((wq_up == nullptr) == (ws_up == nullptr));
  LMOE_ARG_CHECK(xs_pitch >= total_rows);
  if (total_rows == 0) return LMOE_OK;
  LMOE_ARG_CHECK(xq && xs && wq && ws && expert_offsets && output);
  LMOE_ARG_CHECK(aligned16(xq) && aligned16(wq) && aligned16(wq_up));
  LMOE_ARG_CHECK(((reinterpret_cast<uintptr_t>(xs) | reinterpret_cast<uintptr_t>(ws) |
                   reinterpret_cast<uintptr_t>(ws_up)) & 3) == 0);
  LMOE_ARG_CHECK(reinterpret_cast<uintptr_t>(expert_offsets) % (offsets_are_int64 ? 8 : 4) == 0);
  LMOE_ARG_CHECK(reinterpret_cast<uintptr_t>(output) % (out_dtype == LMOE_DTYPE_F32 ? 4 : 2) == 0);
  Fp8Problem p;
  p.xq = xq;
  p.xs = xs;
  p.xs_pitch = xs_pitch;
  p.total_rows = total_rows;
  p.K = K;
  p.wq = wq;
  p.ws = ws;
  p.wq_up = wq_up;
  p.ws_up = ws_up;
  p.N = N;
  p.offsets = expert_offsets;
  p.offsets_i64 = offsets_are_int64;
  p.num_experts = num_experts;
  p.out_dtype = out_dtype;
  p.out = output;
  p.err = error;
  // Few rows: tiles of 256 weight rows stream the weights best (us by rows per expert, that kernel against
  // the other; 8 experts of 4096 x 14336: 1 93 against 132, 64 134 against 137, 96 172 against 137; of 2 x 14336 x 4096:
  // 1 166 against 252, 64 189 against 255, 96 277 against 257; 64 of 2048 x 1408: 1 50 against 75, 64 73 against 77, 96 89
  // against 77; of 2 x 1408 x 2048: 1 80 against 128, 64 110 against 131, 96 141 against 132).  Both give the same bits.  The counts are on
  // the device, so the rule takes all rows.  Uneven loads do not turn it (all rows, that kernel against the other; 4096 rows, 64
  // experts of 2 x 1408 x 2048, the most of one expert 425: 113 against 129, 2048: 107 against 129; 512 rows, 8 of 2 x 14336 x
  // 4096, 106: 209 against 251, 256: 203 against 252; of 4096 x 14336, 106: 127 against 135, 256: 131 against 135), except
  // where one expert has them all, which reads its weights alone and is a short call either way (4096: 78 against 44; 512:
  // 145 against 85).
  return total_rows <= (int64_t)num_experts * kFp8DecodeRows ? run_fp8_decode(p, stream) : run_fp8_gemm(p, stream);
}
