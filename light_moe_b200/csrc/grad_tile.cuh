// grad_tile.cuh -- tiles of the grouped product's gradients (grad_gemm.cu, grad_split.cu).
#pragma once
#include "grad_gemm.h"
#include "host_util.h"
#include "pair_gemm.cuh"

namespace lmoe {

constexpr int kTile = 256, kCta = 128;

struct GradArgs {
  const void* offsets;
  int offsets_i64;
  int E, N, K;       // the product: N is its contraction, K its columns
  int64_t R;
  int MT;            // weight gradient: row tiles of N
  Raster raster;     // of the column tiles of K
  int KS;            // stages of N (not the weight gradient)
  int f16;           // operands fp16 (else bf16)
  void* out;
  int out_dtype;
  int width;         // columns of a tile: 256 or 128
  int splits;        // of the contraction (grad_gemm.cu, not the weight gradient)
  int store;         // StoreMode
  uint32_t* err;
};

struct Tile {
  int e, m, n;
  int row0, row_end;   // input gradient: output rows; weight gradient: the expert's rows
  int ks;              // stages; 0: the tile is zero
};

template <int FORM, int SK>
__device__ __forceinline__ Tile tile_at(const SegTable& t, const GradArgs& a, int tile, int& hint) {
  int j = hint;
  while (tile >= t.tile_start[j + 1]) ++j;
  hint = j;
  Tile r;
  const int rows = t.row[j + 1] - t.row[j];
  a.raster.at(tile - t.tile_start[j], FORM != kGradWeight ? (rows + kTile - 1) / kTile : a.MT, r.m, r.n);
  r.e = j - 1;
  r.row_end = t.row[j + 1];
  if (FORM != kGradWeight) {
    r.row0 = t.row[j] + r.m * kTile;
    r.ks = (j == 0 || j == a.E + 1) ? 0 : a.KS;
  } else {
    r.row0 = t.row[j];
    r.ks = (rows + SK - 1) / SK;
  }
  return r;
}

inline bool weight_grad(const GradProblem& p) { return p.form == kGradWeight; }
// Rows and columns of the second operand.
inline int64_t other_rows(const GradProblem& p) {
  return weight_grad(p) ? p.total_rows : (int64_t)p.num_experts * (p.form == kGradProduct ? p.K : p.N);
}
inline int other_cols(const GradProblem& p) { return p.form == kGradProduct ? p.N : p.K; }
inline int64_t pitch8(int64_t cols) { return (cols + 7) / 8 * 8; }
inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// Rows to copy for TMA: dst rows of `pitch` values from src rows of `cols`.  A call's copies are one
// launch, a job per blockIdx.y.
struct CopyJob {
  const void* src;
  int64_t rows;
  int cols, pitch;
  uint4* dst;
};
struct CopyJobs {
  CopyJob job[2];
  int count;
  void add(const void* src, int64_t rows, int cols, int64_t pitch, void* dst) {
    job[count++] = {src, rows, cols, (int)pitch, static_cast<uint4*>(dst)};
  }
  dim3 grid(const DeviceInfo& dev) const {   // blocks of 256 threads, eight values a thread
    int64_t blocks = 1;
    for (int i = 0; i < count; ++i) {
      const int64_t b = (job[i].rows * (job[i].pitch / 8) + 255) / 256;
      blocks = b > blocks ? b : blocks;
    }
    const int64_t most = (int64_t)dev.num_sms * 8;
    return dim3((unsigned)(blocks < most ? blocks : most), (unsigned)count);
  }
};

// The arguments that both kernels take, and the map of the output's blocks.
inline int fill_args(const GradProblem& p, int sk, int splits, GradArgs& a, CUtensorMap& to) {
  a.offsets = p.offsets;
  a.offsets_i64 = p.offsets_i64;
  a.E = p.num_experts;
  a.N = p.N;
  a.K = p.K;
  a.R = p.total_rows;
  a.MT = (p.N + kTile - 1) / kTile;
  a.KS = (p.N + sk - 1) / sk;
  a.f16 = p.dtype == LMOE_DTYPE_F16;
  a.out = p.out;
  a.out_dtype = p.out_dtype;
  a.store = store_mode(p.out, p.K, p.out_dtype);
  a.err = p.err;
  a.splits = splits;
  if (a.store == kStoreStaged) return LMOE_OK;
  const bool wg = weight_grad(p);
  return encode_store_map(&to, p.out, p.out_dtype, (uint64_t)p.K, wg ? (uint64_t)p.N : (uint64_t)p.total_rows,
                          wg ? (uint64_t)p.num_experts : (uint64_t)splits, 128);
}

}  // namespace lmoe
