// fp4_mma.cuh -- what the two grouped products of 4-bit operands share (fp4_gemm.cu for many rows,
// fp4_decode.cu for few): the block-scaled MMA on a CTA pair, the scale copies to tensor memory,
// and the warps that bring scales into shared memory.
#pragma once
#include "fp4_format.cuh"
#include "fp4_gemm.h"
#include "pair_gemm.cuh"

namespace lmoe {

struct Fp4Args {
  const uint8_t* xs;     // scales of the rows
  int64_t xs_pitch;
  const uint8_t* ws;     // scales of the weights (gate), and of up
  const uint8_t* ws_up;
  int64_t ws_pitch;
  const void* offsets;
  int offsets_i64;
  int E, N, K;
  int64_t R;
  Raster raster;         // of the feature tiles
  int KS;                // stages
  const float* alpha;    // per expert, or NULL
  const float* alpha_up;
  void* out;
  int out_dtype;
  int store;             // StoreMode
  uint32_t* err;
};

struct Fp4Tile {
  int e, m, n, row0, row_end;
  bool zero;   // rows outside every expert
};

template <int ROWS>
__device__ __forceinline__ Fp4Tile fp4_tile_at(const SegTable& t, const Fp4Args& a, int tile, int& hint) {
  int j = hint;
  while (tile >= t.tile_start[j + 1]) ++j;
  hint = j;
  Fp4Tile r;
  const int rows = t.row[j + 1] - t.row[j];
  a.raster.at(tile - t.tile_start[j], (rows + ROWS - 1) / ROWS, r.m, r.n);
  r.e = j - 1;
  r.zero = j == 0 || j == a.E + 1;
  r.row0 = t.row[j] + r.m * ROWS;
  r.row_end = t.row[j + 1];
  return r;
}

constexpr int kFp4Block = 256;   // values of a 128-byte swizzle line of codes
constexpr int kFp4Stage = 512;   // values per stage
// A unit is what one thread issues at a time: four 4-scale words a row; a step two of them.
template <int FORMAT>
struct Fp4Units {
  static constexpr int kUnitK = FORMAT == LMOE_FP4_MX ? 512 : 256;
  static constexpr int kStageUnits = kFp4Stage / kUnitK;
  static constexpr int kStepK = 2 * kUnitK;
};

// Instruction descriptor of the block-scaled kinds: E2M1 operands, K-major, M = 256, N = n.
__host__ __device__ constexpr uint32_t idesc_fp4(bool ue8m0, uint32_t sf_id, uint32_t n) {
  return (sf_id << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((ue8m0 ? 1u : 0u) << 23) |
         ((256u >> 4) << 24) | (sf_id << 29);
}

// Unswizzled descriptor of a 512-byte scale tile (32 rows of 16 bytes).
__device__ __forceinline__ uint64_t sdesc_scales(uint32_t smem_addr) {
  return (uint64_t)((smem_addr >> 4) & 0x3fffu) | ((uint64_t)(128u >> 4) << 32) | ((uint64_t)1u << 46);
}

__device__ __forceinline__ void copy_scales_pair(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

template <int FORMAT>
__device__ __forceinline__ void mma_fp4_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                             uint32_t sfb, uint32_t accumulate) {
  if constexpr (FORMAT == LMOE_FP4_MX)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ float silu(float g) { return __fdividef(g, 1.0f + __expf(-g)); }

// A warp that brings the scales of 64 rows a tile into shared memory: the lane's two rows (rows
// `lane` and `lane + 32`) are words 0, 1 of the 16 bytes at `dst` (the caller adds 8 for the words
// 2, 3 of a 128-row tile).  It reads whole 32-byte sectors, a step (8 words a row, `dst_word` bytes
// apart in the slot) at a time and kAhead steps ahead in registers, and hands a step over with one
// arrival at `full_addr` (+ 8 bytes a slot).  rows(tile, p): the lane's two scale rows of the tile,
// NULL where there is none; false where the tile has no expert.
template <int FORMAT, int SLOTS, typename Rows>
__device__ __forceinline__ void write_scales(int first, int total, int stride, int K, uint8_t* dst, uint32_t dst_word,
                                             uint32_t slot_bytes, uint64_t* sf_empty, uint32_t full_addr,
                                             uint32_t* err, volatile int* abort, uint32_t site, int lane, Rows rows) {
  constexpr int kAhead = 3;
  const int nb = K / fp4_block(FORMAT);
  const int steps = (K + Fp4Units<FORMAT>::kStepK - 1) / Fp4Units<FORMAT>::kStepK;
  int ltile = first, lstep = 0;   // the next load: tile and step
  const uint8_t* lp[2] = {nullptr, nullptr};
  auto next_tile = [&]() {   // first tile at or behind ltile that has an expert
    while (ltile < total && !rows(ltile, lp)) ltile += stride;
  };
  uint32_t v[kAhead][2][8];
  int pending = 0;
  auto load = [&](uint32_t (&b)[2][8]) {
    if (ltile >= total) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int q = 0; q < 8; ++q) b[i][q] = 0u;
      if (lp[i]) ld_global_nc_v8(lp[i] + lstep * 32, b[i]);
    }
    ++pending;
    if (++lstep == steps) {
      lstep = 0;
      ltile += stride;
      next_tile();
    }
  };
  next_tile();
#pragma unroll
  for (int j = 0; j < kAhead; ++j) load(v[j]);
  Ring<SLOTS> sl;
  int step = 0;
  bool ok = true;
  while (ok && pending > 0) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (!ok || pending == 0) break;
      --pending;
      if ((step + 1) * 32 > nb) {
        // scale bytes behind the last block are padding: zero, whatever they hold
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t (&w)[8] = v[j][i];
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const int valid = nb - (step * 32 + q * 4);
            if (valid < 4) w[q] = valid <= 0 ? 0u : (w[q] & ((1u << (8 * valid)) - 1u));
          }
        }
      }
      step = step + 1 == steps ? 0 : step + 1;
      ok = warp_wait(&sf_empty[sl.i], sl.phase ^ 1u, err, abort, site);
      if (!ok) break;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        *reinterpret_cast<uint2*>(dst + sl.i * slot_bytes + q * dst_word) = make_uint2(v[j][0][q], v[j][1][q]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(full_addr + sl.i * 8);
      sl.next();
      load(v[j]);
    }
  }
}

}  // namespace lmoe
