// pair_gemm.cuh -- what the grouped GEMMs on CTA pairs share: the cta_group::2 forms of the
// tcgen05 instructions, cluster barriers, the segment table that every CTA derives from the
// expert offsets, and the row stores of the epilogues.
//
// A pair of CTAs (a cluster of two) computes one tile of 256 rows x BN columns: each CTA holds
// 128 rows of A, half of B's columns in shared memory and 128 x BN accumulators in its tensor
// memory.  One thread of the leader CTA (rank 0) issues the MMAs for both, so each operand
// byte in shared memory feeds twice the work of a single-CTA tile: a 128 x 256 bf16 tile needs
// 96 bytes of operands per SM and cycle from L2 at full tensor rate, a 256 x 256 pair 64.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "grouped_gemm.h"
#include "host_util.h"
#include "lmoe_b200.h"
#include "ptx.cuh"

namespace lmoe {

// The most rows and columns of an operand: the next tile or stage (at most 1024) starts below 2^31.
constexpr int64_t kMaxGemmSize = INT32_MAX - 1024;

// ---------------------------------------------------------------------------------------
// clusters
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Shared-cluster address of `p` (an address of this CTA) in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t mapa_u32(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
// Arrival at a barrier of either CTA.  What it announces is shared or tensor memory of the arriving
// CTA, which only that CTA's tensor core touches next; the caller's proxy fence or tcgen05 fence
// has completed those accesses, so the arrival itself need not order other memory.  (With
// .release.cluster it also waits for the thread's loads and writes to global memory, ~900 ns:
// the 4-bit product of 128 rows took 145 us.)
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// One arrival that also expects `bytes` of copies; it orders no memory (the copies do that).
__device__ __forceinline__ void mbar_arrive_expect_tx_cluster(uint32_t cluster_addr, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], %1;" ::"r"(cluster_addr),
               "r"(bytes)
               : "memory");
}

// Tiled loads into this CTA's shared memory that complete on a barrier of the leader CTA
// (`bar`: its shared-cluster address).  A hand-over by a warp of each CTA would cost an arrival
// with release at cluster scope per stage, which measured ~900 ns (the input gradient of 8192
// rows, N = 14336, K = 4096: 1447 us with the hand-over).
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y,
                                                 int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, "
      "%5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// A producer that gives up leaves its copies a millisecond to land (they take microseconds)
// before its CTA may exit.
__device__ __forceinline__ void let_copies_land() {
  const uint64_t t0 = globaltimer_ns();
  while (globaltimer_ns() - t0 < 1000000ull) {
  }
}

// Position in a ring of N slots and the parity of its pass.
template <int N>
struct Ring {
  uint32_t i = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++i == N) {
      i = 0;
      phase ^= 1u;
    }
  }
};

// The waits of a whole warp, with one answer for all its lanes.  The warps that issue copies and
// MMAs run their loops with all lanes and issue under elect.sync: under `lane == 0` the compiler
// cannot tell that the operands are uniform, and every tcgen05 instruction then costs the thread
// ~60 cycles (measured: the 4-bit product of 16384 rows took 1838 us, 890 cycles of issuer time
// per stage of 384 cycles of MMAs).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, uint32_t* err, volatile int* abort,
                                          uint32_t site) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, abort, site));
}

// ---------------------------------------------------------------------------------------
// tcgen05 on a CTA pair
// ---------------------------------------------------------------------------------------
// One warp of each CTA of the pair executes these.
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)),
               "r"(ncols)
               : "memory");
}
__device__ __forceinline__ void tmem_relinquish_pair() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

__device__ __forceinline__ void mma_ss_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrive once on *bar (the same offset in both CTAs) when all tcgen05 operations that this
// thread issued before have finished.
__device__ __forceinline__ void mma_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}

// The same on a barrier of this CTA alone (the one that issues).
__device__ __forceinline__ void mma_commit_leader(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

// Shared-memory descriptor of an M- or N-major 16-bit operand in 128-byte-swizzled chunks of
// 64 elements x rows: a contraction row is one 128-byte line, eight rows are 1024 bytes, and
// the next 64 elements lie `chunk_bytes` further on.  Sixteen contraction rows advance the
// start address by 2048 bytes.
__device__ __forceinline__ uint64_t sdesc_mn_sw128(uint32_t smem_addr, uint32_t chunk_bytes) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr >> 4) & 0x3fffu);
  d |= (uint64_t)((chunk_bytes >> 4) & 0x3fffu) << 16;   // leading byte offset: the next 64 elements
  d |= (uint64_t)(1024u >> 4) << 32;                     // stride byte offset: the next 8 rows
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)2u << 61;
  return d;
}
constexpr uint32_t kIdescAMajorMN = 1u << 15;
constexpr uint32_t kIdescBMajorMN = 1u << 16;

// Each thread of the warp reads 32 consecutive 32-bit columns of its own TMEM lane.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

// Two of them under one completion wait.
__device__ __forceinline__ void tmem_ld32x2(uint32_t taddr0, uint32_t taddr1, uint32_t (&r)[32], uint32_t (&u)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]),
        "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]),
        "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]),
        "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]),
        "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(taddr0), "r"(taddr1)
      : "memory");
}

// ---------------------------------------------------------------------------------------
// segments
// ---------------------------------------------------------------------------------------
// Row ranges from the expert offsets: segment 0 = rows before the first expert, segment
// 1 + e = expert e, segment E + 1 = rows behind the last expert.  Offsets that decrease or
// leave [0, R] make every expert empty (all rows fall into segment 0), and are reported.
struct SegTable {
  int row[kMaxGemmExperts + 3];          // segment j holds rows [row[j], row[j + 1])
  int tile_start[kMaxGemmExperts + 3];   // first tile of segment j; [segments] = total
  int bad;
};

// Called by all threads of the CTA; `threads` of them.
__device__ __forceinline__ void load_segments(SegTable* t, const void* offsets, int offsets_i64, int E, int64_t R,
                                              int tid, int threads) {
  if (tid == 0) t->bad = 0;
  __syncthreads();
  for (int e = tid; e <= E; e += threads) {
    const int64_t o = offsets_i64 ? static_cast<const int64_t*>(offsets)[e]
                                  : (int64_t) static_cast<const int32_t*>(offsets)[e];
    int64_t prev = 0;
    if (e > 0)
      prev = offsets_i64 ? static_cast<const int64_t*>(offsets)[e - 1]
                         : (int64_t) static_cast<const int32_t*>(offsets)[e - 1];
    if (o < prev || o < 0 || o > R) t->bad = 1;
    t->row[e + 1] = (int)o;
  }
  if (tid == 0) {
    t->row[0] = 0;
    t->row[E + 2] = (int)R;
  }
  __syncthreads();
  if (t->bad)
    for (int e = tid; e <= E; e += threads) t->row[e + 1] = (int)R;
  __syncthreads();
}

// Exclusive scan of the segments' tile counts (count(j) for segment j) by one warp.
template <typename F>
__device__ __forceinline__ void scan_tiles(SegTable* t, int segments, int lane, F count) {
  int carry = 0;
  for (int j0 = 0; j0 < segments; j0 += 32) {
    const int j = j0 + lane;
    int v = j < segments ? count(j) : 0;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    if (j < segments) t->tile_start[j] = carry + s - v;
    carry += __shfl_sync(0xffffffffu, s, 31);
  }
  if (lane == 0) t->tile_start[segments] = carry;
}

// Tile `local` of a segment of mt x nb tiles.  Tiles are walked in groups of eight row tiles,
// column tile by column tile inside a group, so that the pairs working at the same time share
// eight row panels and a few column panels through L2.  Every role of the kernel walks the tiles
// by itself, the MMA issuer between the MMAs of two tiles, so the two divisions are
// multiplications (with them: ~1000 cycles a tile).
struct Raster {
  int nb, per;      // column tiles; tiles of a full group
  uint32_t magic;   // floor(2^32 / per)
  __host__ __device__ Raster(int nb_ = 1)
      : nb(nb_), per(8 * nb_), magic((uint32_t)(0x100000000ull / (uint32_t)(8 * nb_))) {}
  // ceil(2^32 / d) of 2 .. 7
  static __device__ __forceinline__ uint32_t small_magic(int d) {
    return d < 4 ? (d == 2 ? 0x80000000u : 0x55555556u)
                 : (d < 6 ? (d == 4 ? 0x40000000u : 0x33333334u) : (d == 6 ? 0x2aaaaaabu : 0x24924925u));
  }
  __device__ __forceinline__ void at(int local, int mt, int& m, int& n) const {
    // the product is below the quotient by less than one
    int g = (int)__umulhi((uint32_t)local, magic);
    int in = local - g * per;
    if (in >= per) {
      ++g;
      in -= per;
    }
    const int gm = mt - g * 8;
    if (gm >= 8) {
      n = in >> 3;
      m = g * 8 + (in & 7);
    } else {
      // ceil(2^32 / gm) is exact for in * gm < 2^32
      const uint32_t q = gm == 1 ? (uint32_t)in : __umulhi((uint32_t)in, small_magic(gm));
      n = (int)q;
      m = g * 8 + in - (int)q * gm;
    }
  }
};

// ---------------------------------------------------------------------------------------
// epilogue stores
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t pack16(float a, float b, int f16) {
  if (f16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// How rows of an output can be stored: whole 32-byte sectors, 16-byte vectors, or neither.
enum StoreMode : int { kStoreStaged = 0, kStore16 = 16, kStore32 = 32 };
inline int store_mode(const void* out, int64_t cols, int dtype) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(out) | (uintptr_t)(cols * (dtype == LMOE_DTYPE_F32 ? 4 : 2));
  return a % 32 == 0 ? kStore32 : (a % 16 == 0 ? kStore16 : kStoreStaged);
}
// Called by a whole warp: lane l holds COLS values of row l (of `rows` valid ones) from column c0;
// columns at or behind `cols` are not written.  Rows that do not start at whole vectors go through
// `stage` (STAGE bytes of the warp's own), so that neighbouring lanes write neighbouring columns, up
// to 128 bytes of a row at a time: storing them value by value from the lanes that hold them touches
// 32 sectors per instruction (the gradients of fp16 rows of odd lengths took 7.9 ms, of which ~7 ms
// stores).
template <int COLS, uint32_t STAGE>
__device__ __forceinline__ void store_rows(uint8_t* base, int64_t pitch, int rows, int c0, int cols,
                                           const float (&v)[COLS], int dtype, int mode, uint8_t* stage, int lane) {
  if (c0 >= cols || rows <= 0) return;
  const bool f16 = dtype == LMOE_DTYPE_F16;
  if (mode != kStoreStaged) {
    if (lane >= rows) return;
    uint8_t* row = base + lane * pitch;
    if (dtype == LMOE_DTYPE_F32) {
      float* p = reinterpret_cast<float*>(row) + c0;
#pragma unroll
      for (int j = 0; j < COLS / 8; ++j) {
        if (mode == kStore32 && c0 + 8 * j < cols) {
          uint32_t w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[8 * j + i]);
          st_global_v8(p + 8 * j, w);
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (c0 + 8 * j + 4 * i < cols)
              *reinterpret_cast<float4*>(p + 8 * j + 4 * i) =
                  make_float4(v[8 * j + 4 * i], v[8 * j + 4 * i + 1], v[8 * j + 4 * i + 2], v[8 * j + 4 * i + 3]);
        }
      }
    } else {
      uint16_t* p = reinterpret_cast<uint16_t*>(row) + c0;
#pragma unroll
      for (int j = 0; j < COLS / 16; ++j) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = pack16(v[16 * j + 2 * i], v[16 * j + 2 * i + 1], f16);
        if (mode == kStore32 && c0 + 16 * j < cols) {
          st_global_v8(p + 16 * j, w);
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (c0 + 16 * j + 8 * i < cols)
              *reinterpret_cast<uint4*>(p + 16 * j + 8 * i) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        }
      }
    }
    return;
  }
  // W words of a row at a time, word j of row r at j ^ r (mod W)
  constexpr int kUnroll = COLS == 64 ? 1 : 4;   // 64 values leave no registers for more
  uint32_t* st = reinterpret_cast<uint32_t*>(stage);
  if (dtype == LMOE_DTYPE_F32) {
    constexpr int W = COLS < (int)STAGE / 128 ? COLS : (int)STAGE / 128;
    static_assert((W & (W - 1)) == 0 && W <= 32 && COLS % W == 0, "words of a row");
#pragma unroll
    for (int ch = 0; ch < COLS / W; ++ch) {
#pragma unroll
      for (int i = 0; i < W; ++i) st[lane * W + ((i ^ lane) & (W - 1))] = __float_as_uint(v[W * ch + i]);
      __syncwarp();
      const int j = lane & (W - 1), c = c0 + W * ch + j;
      if (c < cols)
#pragma unroll kUnroll
        for (int r = lane / W; r < rows; r += 32 / W)
          reinterpret_cast<uint32_t*>(base + r * pitch)[c] = st[r * W + ((j ^ r) & (W - 1))];
      __syncwarp();
    }
  } else {
    constexpr int W = COLS / 2 < (int)STAGE / 128 ? COLS / 2 : (int)STAGE / 128;
    static_assert((W & (W - 1)) == 0 && W <= 32 && COLS % (2 * W) == 0, "words of a row");
    const bool pairs = ((reinterpret_cast<uintptr_t>(base) | (uintptr_t)pitch) & 3) == 0;   // rows of whole words
#pragma unroll
    for (int ch = 0; ch < COLS / (2 * W); ++ch) {
#pragma unroll
      for (int i = 0; i < W; ++i)
        st[lane * W + ((i ^ lane) & (W - 1))] = pack16(v[2 * (W * ch + i)], v[2 * (W * ch + i) + 1], f16);
      __syncwarp();
      const int at = c0 + 2 * W * ch;
      if (pairs) {
        const int j = lane & (W - 1), c = at + 2 * j;
        if (c < cols)
#pragma unroll kUnroll
          for (int r = lane / W; r < rows; r += 32 / W)
            *reinterpret_cast<uint32_t*>(base + r * pitch + c * 2) = st[r * W + ((j ^ r) & (W - 1))];
      } else {
        constexpr int P = W < 16 ? 2 * W : 32;   // values of a row at a time
#pragma unroll kUnroll
        for (int h = 0; h < 2 * W / P; ++h) {
          const int k = h * P + (lane & (P - 1)), c = at + k, j = k >> 1;
          if (c < cols)
#pragma unroll kUnroll
            for (int r = lane / P; r < rows; r += 32 / P)
              reinterpret_cast<uint16_t*>(base + r * pitch)[c] =
                  (uint16_t)(st[r * W + ((j ^ r) & (W - 1))] >> (16 * (k & 1)));
        }
      }
      __syncwarp();
    }
  }
}

// A block of a warp's 32 rows x LINE bytes (lane l: row l; LINE / 2 16-bit values or LINE / 4 of fp32
// from v) into `stage`, in the LINE-byte swizzle of the output's tensor map, ready for a tiled
// store.  (The lanes' own 32-byte stores, each to another row, keep the L1 data pipe busy ~54 cycles
// per instruction: 62 % of the kernel in a weight gradient of short segments.)
template <int LINE>
__device__ __forceinline__ void stage_block(const float* v, int dtype, uint8_t* stage, int lane) {
  uint8_t* row = stage + lane * LINE;
  const int x = LINE == 128 ? lane & 7 : LINE == 64 ? (lane >> 1) & 3 : (lane >> 2) & 1;   // 16-byte piece j of the row lies at j ^ x
#pragma unroll
  for (int j = 0; j < LINE / 16; ++j) {
    uint4 w;
    if (dtype == LMOE_DTYPE_F32) {
      w = make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]),
                     __float_as_uint(v[4 * j + 3]));
    } else {
      const bool f16 = dtype == LMOE_DTYPE_F16;
      w = make_uint4(pack16(v[8 * j], v[8 * j + 1], f16), pack16(v[8 * j + 2], v[8 * j + 3], f16),
                     pack16(v[8 * j + 4], v[8 * j + 5], f16), pack16(v[8 * j + 6], v[8 * j + 7], f16));
    }
    *reinterpret_cast<uint4*>(row + ((j ^ x) * 16)) = w;
  }
}
// The block's way out: called by the whole warp; `stage` must not be read by an earlier store.
template <int LINE>
__device__ __forceinline__ void store_block(const CUtensorMap* map, const float* v, int dtype, uint8_t* stage,
                                            int lane, int x, int y, int z) {
  if (elect_one()) bulk_wait_read();
  __syncwarp();
  stage_block<LINE>(v, dtype, stage, lane);
  fence_proxy_async_smem();
  __syncwarp();
  if (elect_one()) {
    tma_store_3d(map, stage, x, y, z);
    bulk_commit();
  }
  __syncwarp();
}
// The tensor map of an output [count][rows][cols] for blocks of `line` bytes x 32 rows.
inline int encode_store_map(CUtensorMap* map, const void* out, int dtype, uint64_t cols, uint64_t rows, uint64_t count,
                            uint32_t line) {
  const uint32_t es = dtype == LMOE_DTYPE_F32 ? 4 : 2;
  const CUtensorMapDataType dt = dtype == LMOE_DTYPE_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : dtype == LMOE_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                           : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint64_t dims[3] = {cols, rows, count}, strides[2] = {cols * es, cols * es * rows};
  const uint32_t box[3] = {line / es, 32, 1};
  return encode_tmap_3d(map, out, dt, es, dims, strides, box);
}

// Width of the column tiles: the one with the shortest static schedule of `tiles(width)` tiles on
// `pairs` pairs, a round taking as long as its columns and a constant (`floor_cols`: what a
// round costs at least, `extra`: what a tile costs beside its columns).  With few rows a kernel
// streams weights, and the last round of wide tiles leaves most pairs idle.
template <int N, typename F>
inline int pick_width(const int (&widths)[N], int pairs, int floor_cols, int extra, F tiles) {
  int best = widths[0];
  int64_t best_cost = INT64_MAX;
  for (int w : widths) {
    const int64_t rounds = (tiles(w) + pairs - 1) / pairs;
    const int64_t cost = rounds * ((w > floor_cols ? w : floor_cols) + extra);
    if (cost < best_cost) {
      best_cost = cost;
      best = w;
    }
  }
  return best;
}
// Row tiles of `rows` rows spread evenly over `experts` experts (the counts are on the device).
inline int64_t even_row_tiles(int64_t rows, int experts, int tile) {
  if (rows <= experts) return rows;
  const int64_t each = (rows + experts - 1) / experts;
  return (each + tile - 1) / tile * experts;
}

}  // namespace lmoe
