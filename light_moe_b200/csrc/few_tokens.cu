// few_tokens.cu -- a whole MoE layer for up to 16 tokens in two kernels (sm_100a).
//
//   p = softmax(x G^T + bias), the k most probable experts (ties to the lower id), w = p / sum of theirs
//   y[t] = sum_j w[t, j] * W2[e_j] (silu(W1[e_j] x[t]) * (W3[e_j] x[t]))  + the same of every shared expert, w = 1
//
// Weights dense (the tokens' 16-bit type) or E4M3 with a scale per 128 x 128 block (fp8_format.cuh).  A
// few tokens read every weight of their experts once and do a few operations with it: the kernels
// are bound by HBM, and what they have to do is keep enough loads in flight and spend few
// instructions on a weight.
//
// Warps load weights straight into the fragments of mma.sync.m16n8k16, whose 16 rows are weight rows
// and whose 8 columns are tokens: which contraction index a lane's register stands for is free as
// long as both operands agree, so a lane takes 32 consecutive bytes of a row (the quad of a row 128)
// and no weight passes through shared memory.  One instruction multiplies 256 weights with all
// tokens, against 256 x tokens / 32 multiply-adds on the CUDA cores; a 5th-generation MMA would
// want its operands in shared memory, which costs more than it gives for 8 columns.  E4M3 values are
// exact in fp16.
//
// An expert that some token chose is multiplied with a whole fragment of tokens, since columns are free: with up to 8
// tokens the first kernel takes all of them and drops the results of those that did not choose the expert; with more,
// and with more than 4 in the second kernel, the expert's own tokens are packed into the fragment's columns.  There is
// no permutation, and the second kernel is one product over the contraction (expert, hidden feature) whose sum is the
// weighted combine.
//
// 1. gate_up_kernel.  Every CTA computes the routing for itself (a few microseconds of L2 reads; a
//    kernel of its own would cost more), then the CTAs share the tiles of 8 hidden features: rows 0-7
//    of an MMA are gate rows and rows 8-15 the same rows of up, so one thread holds gate and up of
//    a feature.  The 16 warps of a CTA split a tile's contraction and join it in shared memory.
//    Writes w * silu(gate) * up in fp32.
// 2. down_kernel.  A CTA owns 256 output rows (a warp 16) and a slice of the contraction; the last
//    CTA of a row block to finish adds the slices in their order, so the result does not depend on
//    timing.  Hidden values enter the MMA as a sum of two fp16 numbers (22 bits) or three bf16 numbers (all 24), which
//    cost columns of the MMA (8 hold 4 tokens, or 2) but no weight traffic: rounding them to one would be an error
//    as large as the output's own rounding, and with two bf16 numbers (16 bits) 0.28 % of a layer's outputs lay on the
//    other side of a bf16 step than in exact arithmetic, with three 0.04 %, in fp32 arithmetic 0.06 % (4 tokens, 8
//    experts of 4096 x 14336; 318 us with two, 323 with three).
//
// fp16 operands need a range: tokens (bf16 times E4M3 weights) and hidden values are scaled by powers of two, per token
// (hidden values over all of its experts), so that the largest lies in [2^14, 2^15); what is 2^-39 of it or smaller is
// lost.
//
// Measured, whole calls, us: one token, E4M3, 2 of 8 experts of 4096 x 14336: 78 (352 MB of weights: 4.5 TB/s; the
// routing, the joins and the two kernels' ramps take 22 us); 4 tokens, bf16, 5 or 6 experts of the same layer, 1.8-2.1 GB:
// 309-331, 5.7-6.4 TB/s; 16 tokens, E4M3, all 8 experts, 1.41 GB: 403; one token, fp16, 2 of 8 experts of 1024 x 2816:
// 22.5, which is latency: two launches, a router, three joins.  First / second kernel apart, from cold caches under a
// profiler: one token, E4M3 54 / 31; 16 tokens, E4M3 241 / 152; 4 tokens, bf16, 4 experts (1.41 GB) 148 / 91.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "fp8_format.cuh"
#include "host_util.h"
#include "lmoe_math.cuh"
#include "ptx.cuh"

namespace lmoe {
namespace {

constexpr int kWarps = 16, kThreads = kWarps * 32;
constexpr int kMaxTokens = 16, kMaxExperts = 256, kMaxShared = 16, kMaxTopK = 16;
constexpr int kMaxUsed = kMaxExperts + kMaxShared;
// Steps of weights in flight per warp (4 of E4M3 cost registers: 85.5 us for 78.6, one token, 8 experts of 4096 x 14336).
template <bool FP8>
constexpr int kAheadOf = FP8 ? 3 : 4;
// The second kernel's warps each read rows of their own, and ask for two or three steps of a row at a time: 128
// bytes here and there open as many pages of the memory (4 tokens, bf16, the same layer, when this was chosen: 130 us of it
// step by step, 112 so).
constexpr int kRowBlock = kWarps * 16;   // output rows of a CTA of the second kernel
constexpr int kSplitCtas = 148;  // CTAs that the second kernel's slices aim at: one per SM, whatever the limit of CTAs
constexpr int kMaxCtas = 256;    // of the first kernel
constexpr int kJoins = 4;        // tiles whose parts may wait to be joined
// Hidden values in shared memory at a time: a slice's, if they fit kWholeBytes, else chunks of a multiple of
// kChunkSteps steps in two buffers of kStageBytes (of 12 steps at least: 96 KB for 16 tokens).  What shared memory
// takes is missing in L1, through which the weights' loads go: with 200 KB the second kernel read bf16 weights at 4.3
// TB/s (149 us of 4 tokens, 8 experts of 4096 x 14336, two terms to a hidden value), so at 6.2 (103 us).  Three terms to a
// value take half as much again, and chunks cost them more than L1 does (7 tokens, 64 experts of 1408 x 2048 and two
// shared: 166 us in chunks, 160 whole).
constexpr int kChunkSteps = 12;
constexpr uint32_t kStageBytes = 64 * 1024, kWholeBytes = 128 * 1024, kWholeBytes3 = 176 * 1024;
constexpr uint32_t kSite = 0x800u;
constexpr float kInf = __builtin_huge_valf();

// What the first kernel tells the second.
struct Header {
  uint32_t error;            // of the kernels' waits
  int used;                  // experts with tokens
  int pad[2];
  int expert[kMaxUsed];      // ascending, shared ones last
  uint32_t tokens[kMaxUsed]; // bit t: token t chose it
};

struct FewArgs {
  const void* x;             // [T, d]
  const void* gate;          // [E, d]
  const float* bias;
  const uint8_t* w1;         // [E + S, F, d]
  const uint8_t* w3;
  const uint8_t* w2;         // [E + S, d, F]
  const float* s1;           // block scales (fp8)
  const float* s3;
  const float* s2;
  int T, d, F, E, k, S;
  int groups;                // token groups of the first kernel
  int split;                 // slices of the second kernel
  int grid1;                 // CTAs of the first
  int item0;                 // row block and slice of the second kernel's first CTA
  int chunk;                 // steps of hidden values that the second stages at a time
  uint32_t sums_at;          // offset of its tokens' sums in shared memory
  void* y;
  int32_t* ids;
  float* weights;
  Header* head;
  uint32_t* counters;        // arrivals per row block
  uint32_t* tops;            // [CTA of the first kernel][T]: fp32 bits of its largest hidden value
  float* h;                  // [used][T][F]
  float* part;               // [split][T][d]
};

// A weight row's 32 bytes per lane and step.
template <bool FP8>
struct Geo {
  static constexpr int kPer = FP8 ? 32 : 16;      // values of a lane
  static constexpr int kStep = 4 * kPer;          // values of a step: of the quad of a row
  static constexpr int kPieces = kPer / 8;        // 16-byte pieces (8 values) of the 16-bit operand
  static constexpr int kBytes = FP8 ? 1 : 2;
};

// 16-bit numbers whose sum a hidden value is in the second kernel: of 11 significant bits, or of 8.
template <bool FP8, typename X>
constexpr int kTermsOf = !FP8 && std::is_same<X, __nv_bfloat16>::value ? 3 : 2;

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two rows' 32 bytes (rows g and g + 8 of the MMA) times piece p of the other operand.
template <bool FP8, typename M>
__device__ __forceinline__ void mma_piece(float (&c)[4], const uint32_t (&lo)[8], const uint32_t (&hi)[8], int p,
                                          const uint4& b) {
  if constexpr (FP8) {
    mma16816<M>(c, e4m3x2_half2(lo[2 * p]), e4m3x2_half2(hi[2 * p]), e4m3x2_half2_high(lo[2 * p]),
                e4m3x2_half2_high(hi[2 * p]), b.x, b.y);
    mma16816<M>(c, e4m3x2_half2(lo[2 * p + 1]), e4m3x2_half2(hi[2 * p + 1]), e4m3x2_half2_high(lo[2 * p + 1]),
                e4m3x2_half2_high(hi[2 * p + 1]), b.z, b.w);
  } else {
    mma16816<M>(c, lo[4 * p], hi[4 * p], lo[4 * p + 1], hi[4 * p + 1], b.x, b.y);
    mma16816<M>(c, lo[4 * p + 2], hi[4 * p + 2], lo[4 * p + 3], hi[4 * p + 3], b.z, b.w);
  }
}

// Offset of the 16-byte piece with values 8 * q .. 8 * q + 7 of token t in an operand of `tokens` tokens:
// [step][piece][token][lane of the quad], so that a quarter warp reads 128 consecutive bytes.
template <bool FP8>
__device__ __forceinline__ uint32_t piece_offset(int q, int t, int tokens) {
  using G = Geo<FP8>;
  const int step = q / (G::kStep / 8), in = q % (G::kStep / 8);
  return (((uint32_t)step * G::kPieces + in % G::kPieces) * tokens + t) * 64 + in / G::kPieces * 16;
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 .. 127

// Exponent that brings the largest absolute value (its fp32 bits, finite) to [2^14, 2^15).
__device__ __forceinline__ int range_exponent(uint32_t top) {
  if (top == 0) return 0;
  const int e = 14 - ((int)(top >> 23) - 127);   // subnormals count as 2^-127
  return e > 126 ? 126 : e;
}

template <typename T>
__device__ __forceinline__ float2 widen2(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value)
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
// fp32 bits of the largest finite absolute value of a 16-bit pair.
template <typename T>
__device__ __forceinline__ uint32_t finite_top(uint32_t w) {
  const float2 v = widen2<T>(w);
  const uint32_t a = __float_as_uint(v.x) & 0x7fffffffu, b = __float_as_uint(v.y) & 0x7fffffffu;
  return max(a < 0x7f800000u ? a : 0u, b < 0x7f800000u ? b : 0u);
}

__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Shared-cluster address of `p` (an address of this CTA) in CTA `rank` of the cluster, and a load from there.
__device__ __forceinline__ uint32_t mapa_u32(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// The second kernel is launched while the first one runs: its CTAs start as the first one's leave
// their SMs, and wait here for all of it.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_launcher() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---------------------------------------------------------------------------------------
// first kernel
// ---------------------------------------------------------------------------------------
struct FewShared {
  uint32_t used_tokens[kMaxUsed];   // bit t: token t chose expert e (all experts)
  int list[kMaxUsed];               // experts with tokens
  int group[kMaxUsed];              // positions in `list` that have tokens of the group
  int used, group_used, warps_per_tile;
  uint64_t full[kJoins][kWarps];    // a tile's parts are written (its warps)
  uint64_t empty[kJoins][kWarps];   // ... and joined
  int abort;
  uint32_t htop[kMaxTokens];        // largest hidden values
  uint32_t top[kMaxTokens];         // largest absolute value of the group's tokens
  float unscale[kMaxTokens];
  uint8_t column[kMaxUsed][kMaxTokens];   // of more than 8 tokens: those of an expert, one after the other
};

// Dynamic shared memory of the first kernel.
struct FewLayout {
  uint32_t x, red, share, total;
};
__host__ __device__ inline FewLayout few_layout(int d, int step, int group_tokens, int T, int experts) {
  FewLayout l;
  const uint32_t kpad = (uint32_t)(d + step - 1) / step * step;
  const uint32_t nt = group_tokens > 8 ? 2 : 1;
  l.x = 0;
  l.red = kpad * group_tokens * 2;
  l.share = l.red + kJoins * kWarps * 16 * 8 * nt * 4;
  l.total = l.share + (uint32_t)(experts * T + 3) / 4 * 16;
  return l;
}

template <bool FP8, typename X, int NT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) gate_up_kernel(const FewArgs a) {
  using G = Geo<FP8>;
  using M = typename std::conditional<FP8, __half, X>::type;   // type of the products
  constexpr int kAhead = kAheadOf<FP8>;
  constexpr bool kScaled = FP8 && std::is_same<X, __nv_bfloat16>::value;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ FewShared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int steps = (a.d + G::kStep - 1) / G::kStep;
  const int per_group = a.groups == 1 ? a.T : 8;
  const int experts = a.E + a.S;
  const FewLayout lay = few_layout(a.d, G::kStep, per_group, a.T, experts);
  float* red = reinterpret_cast<float*>(smem + lay.red);
  float* share = reinterpret_cast<float*>(smem + lay.share);     // [E + S][T]: routing weights
  constexpr int kRedRow = 8 * NT, kRedWarp = 16 * kRedRow, kRedBuf = kWarps * kRedWarp;
  float* logits = red + kRedBuf;   // [tokens of the group][256], while routing
  float* halves = logits + 8 * NT * kMaxExperts;   // a CTA's share of them
  static_assert((kJoins - 1) * kRedBuf >= 2 * 8 * NT * kMaxExperts, "room for the logits");
  const int pieces = steps * G::kStep / 8;   // of a token; behind d: zeros
  launch_dependents();

  // The router's weights are 16 experts a fragment; warps that have the same one share its steps, and with many
  // experts the two CTAs of a pair do: all CTAs read them at the same time, which L2 feeds at its own rate (64
  // experts of 2048: 7 tokens 96 us replayed, 88.5 shared).  The first two steps' loads start before the tokens
  // are there.
  const uint32_t rank = cluster_ctarank();
  const int shares = a.E > 16 ? 2 : 1, lead = shares == 2 ? (int)rank : 0;   // steps lead, lead + shares, ...
  const int mtiles = (a.E + 15) / 16;
  const int wpm = mtiles == 1 ? 16 : (mtiles == 2 ? 8 : (mtiles <= 4 ? 4 : (mtiles <= 8 ? 2 : 1)));
  const int e0 = warp / wpm * 16;
  const X* r0 = static_cast<const X*>(a.gate) + (int64_t)(e0 + g) * a.d + c * G::kPer;
  const X* r1 = r0 + (int64_t)8 * a.d;
  auto load_gate = [&](int s, uint4 (&v0)[G::kPieces], uint4 (&v1)[G::kPieces]) {
#pragma unroll
    for (int p = 0; p < G::kPieces; ++p) {
      const int at = s * G::kStep + p * 8;
      const bool in = at + c * G::kPer < a.d && s < steps;
      v0[p] = v1[p] = make_uint4(0u, 0u, 0u, 0u);
      if (in && e0 + g < a.E) v0[p] = __ldg(reinterpret_cast<const uint4*>(r0 + at));
      if (in && e0 + g + 8 < a.E) v1[p] = __ldg(reinterpret_cast<const uint4*>(r1 + at));
    }
  };

  if (tid < kMaxTokens) {
    sh.htop[tid] = 0u;
    sh.top[tid] = 0u;
  }
  if (tid == 0) sh.abort = 0;
  if (tid == 0 && blockIdx.x == 0) a.head->error = 0u;
  for (int i = tid; i < experts * a.T; i += kThreads) share[i] = i >= a.E * a.T ? 1.0f : 0.0f;
  for (int e = tid; e < experts; e += kThreads) sh.used_tokens[e] = e >= a.E ? (1u << a.T) - 1u : 0u;

  // tokens t0 .. t0 + n - 1 into shared memory, in the order of the fragments
  auto load_x = [&](int t0, int n) {
    __syncthreads();   // earlier readers of the tokens, and their largest values set to 0
    for (int i0 = warp * 32; i0 < pieces * n; i0 += kThreads) {
      const int i = i0 + lane, t = n == 1 ? 0 : i / pieces, q = i - t * pieces;
      uint32_t m = 0u;
      if (t < n && q < pieces) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (q * 8 < a.d) v = __ldg(reinterpret_cast<const uint4*>(static_cast<const X*>(a.x) + (int64_t)(t0 + t) * a.d) + q);
        *reinterpret_cast<uint4*>(smem + lay.x + piece_offset<FP8>(q, t, n)) = v;
        if (kScaled) m = max(max(finite_top<X>(v.x), finite_top<X>(v.y)), max(finite_top<X>(v.z), finite_top<X>(v.w)));
      }
      if (kScaled) {
        const uint32_t same = __match_any_sync(0xffffffffu, t);
        const uint32_t most = __reduce_max_sync(same, m);
        if (t < n && lane == __ffs(same) - 1) atomicMax(&sh.top[t], most);
      }
    }
    __syncthreads();
  };
  // ... and to scaled fp16 in place, by the warps from `first` on
  auto scale_x = [&](int n, int first) {
    if constexpr (kScaled) {
      if (warp < first) return;
      for (int i = tid - first * 32; i < pieces * n; i += kThreads - first * 32) {
        const int t = n == 1 ? 0 : i / pieces, q = i - t * pieces;
        const float f = pow2(range_exponent(sh.top[t]));
        uint4* p = reinterpret_cast<uint4*>(smem + lay.x + piece_offset<FP8>(q, t, n));
        uint4 v = *p;
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f2 = widen2<X>(w[j]);
          w[j] = narrow2<M>(f2.x * f, f2.y * f);
        }
        *p = v;
      }
      if (warp == first && lane < n) sh.unscale[lane] = pow2(-range_exponent(sh.top[lane]));
    }
  };
  if (!kScaled && tid < kMaxTokens) sh.unscale[tid] = 1.0f;

  // ---- routing
  for (int t0 = 0; t0 < a.T; t0 += per_group) {
    const int n = a.T - t0 < per_group ? a.T - t0 : per_group;
    uint4 v[2][2][G::kPieces];
    const int s_first = warp % wpm * shares + lead, s_step = wpm * shares;
    load_gate(s_first, v[0][0], v[0][1]);
    load_gate(s_first + s_step, v[1][0], v[1][1]);
    load_x(t0, n);
    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
    for (int s0 = s_first; s0 < steps; s0 += 2 * s_step) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int s = s0 + b * s_step;
        if (s >= steps) break;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          const int t = i * 8 + g;
#pragma unroll
          for (int p = 0; p < G::kPieces; ++p) {
            uint4 x = make_uint4(0u, 0u, 0u, 0u);
            if (t < n) x = *reinterpret_cast<const uint4*>(smem + lay.x + ((uint32_t)(s * G::kPieces + p) * n + t) * 64 + c * 16);
            mma16816<X>(part, v[b][0][p].x, v[b][1][p].x, v[b][0][p].y, v[b][1][p].y, x.x, x.y);
            mma16816<X>(part, v[b][0][p].z, v[b][1][p].z, v[b][0][p].w, v[b][1][p].w, x.z, x.w);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] += part[j];
        }
        load_gate(s + 2 * s_step, v[b][0], v[b][1]);
      }
    }
    float* mine = red + warp * kRedWarp;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      *reinterpret_cast<float2*>(mine + g * kRedRow + i * 8 + c * 2) = make_float2(acc[i][0], acc[i][1]);
      *reinterpret_cast<float2*>(mine + (g + 8) * kRedRow + i * 8 + c * 2) = make_float2(acc[i][2], acc[i][3]);
    }
    __syncthreads();
    if (shares == 2) {
      for (int i = tid; i < n * a.E; i += kThreads) {
        const int t = n == 1 ? 0 : i / a.E, e = i - t * a.E;
        const float* r = red + (e >> 4) * wpm * kRedWarp + (e & 15) * kRedRow + t;
        float sum = 0.0f;
#pragma unroll 4
        for (int w = 0; w < wpm; ++w) sum += r[w * kRedWarp];
        halves[t * kMaxExperts + e] = sum;
      }
      cluster_sync();
    }
    if (warp < n) {
      // One warp per token.  A pick is the best one behind the last pick, in the order of logits and ids
      // (little code: what runs once waits for its instructions).
      const int t = warp;
      float* mine_l = logits + t * kMaxExperts;
      auto sum_parts = [&](int e) {
        const float* r = red + (e >> 4) * wpm * kRedWarp + (e & 15) * kRedRow + t;
        float sum = 0.0f;
#pragma unroll 4
        for (int w = 0; w < wpm; ++w) sum += r[w * kRedWarp];
        return sum;
      };
      for (int e = lane; e < a.E; e += 32) {
        float sum;
        if (shares == 2) {   // the CTAs' halves, in the order of their ranks
          const float mine = halves[t * kMaxExperts + e], other = ld_cluster(mapa_u32(&halves[t * kMaxExperts + e], rank ^ 1u));
          sum = rank == 0 ? mine + other : other + mine;
        } else {
          sum = sum_parts(e);
        }
        mine_l[e] = a.bias ? sum + __ldg(a.bias + e) : sum;
      }
      float top = 0.0f, sum = 0.0f, mine_p = 0.0f;
      int chosen = 0, last = -1;
      uint32_t last_key = 0xffffffffu;
#pragma unroll 1
      for (int j = 0; j < a.k; ++j) {
        uint32_t key = 0u;   // orders like the logits; NaN lowest, 0: none
        int at = kMaxExperts;
        float l = 0.0f;
#pragma unroll 1
        for (int e = lane; e < a.E; e += 32) {
          const float v = mine_l[e];
          const uint32_t b = __float_as_uint(v);
          const uint32_t k = v == v ? ((b & 0x80000000u) ? ~b : (b | 0x80000000u)) : 1u;
          if ((k < last_key || (k == last_key && e > last)) && k > key) {
            key = k;
            at = e;
            l = v;
          }
        }
        last_key = __reduce_max_sync(0xffffffffu, key);
        last = (int)__reduce_min_sync(0xffffffffu, key == last_key ? (unsigned)at : (unsigned)kMaxExperts);
        l = __shfl_sync(0xffffffffu, l, last & 31);
        if (j == 0) top = l;
        // (a NaN, and what has no softmax: nothing but -inf, or +inf)
        const float p = l == l && fabsf(top) < kInf ? softmax_exp(l - top) : __uint_as_float(0x7fc00000u);
        sum += p;
        if (lane == j) {
          mine_p = p;
          chosen = last;
        }
      }
      if (lane < a.k) {
        const float w = __fdiv_rn(mine_p, sum);
        share[chosen * a.T + t0 + t] = w;
        atomicOr(&sh.used_tokens[chosen], 1u << (t0 + t));
        if (blockIdx.x == 0) {
          a.ids[(t0 + t) * a.k + lane] = chosen;
          a.weights[(t0 + t) * a.k + lane] = w;
        }
      }
    }
    // the warps without a token meanwhile
    if (a.groups == 1) scale_x(n, n < kWarps ? n : 0);
    if (a.groups > 1 && tid < kMaxTokens) sh.top[tid] = 0u;
    if (shares == 2)
      cluster_sync();   // the other CTA has read this one's share
    else
      __syncthreads();
  }

  // ---- the used experts, and the warps of a tile: a power of two, each with a step at least.  Many balance
  // the last round, few have less to join (half a step's time a tile).  Reckoned for all SMs whatever the grid:
  // the order of the sums, and so their last bits, do not depend on a limit of CTAs.
  const int ftiles = a.F / 8;
  if (warp == 0) {
    int n = 0;
    for (int b0 = 0; b0 < experts; b0 += 32) {
      const int e = b0 + lane;
      const bool used = e < experts && sh.used_tokens[e] != 0u;
      const uint32_t m = __ballot_sync(0xffffffffu, used);
      const int at = n + __popc(m & ((1u << lane) - 1u));
      if (used) {
        sh.list[at] = e;
        sh.group[at] = at;
        if (NT > 1) {
          uint32_t left = sh.used_tokens[e];
          for (int j = 0; left; ++j, left &= left - 1u) sh.column[at][j] = (uint8_t)(__ffs(left) - 1);
        }
      }
      n += __popc(m);
    }
    const int w = 1 << lane, groups = kSplitCtas * kWarps >> lane;   // lanes 0 .. 4
    unsigned cost = 0xffffffffu;
    if (lane < 5 && w <= steps)
      cost = (unsigned)((n * ftiles + groups - 1) / groups * (2 * ((steps + w - 1) >> lane) + 1)) << 3 | lane;
    const int wpt = 1 << (__reduce_min_sync(0xffffffffu, cost) & 7u);
    if (lane == 0) {
      sh.used = sh.group_used = n;
      sh.warps_per_tile = wpt;
    }
    for (int i = lane; i < kJoins * kWarps; i += 32) {
      mbar_init(&sh.full[i / kWarps][i % kWarps], (uint32_t)wpt);
      mbar_init(&sh.empty[i / kWarps][i % kWarps], 1);
    }
    fence_mbar_init();
  }
  __syncthreads();

  // ---- the experts' gate and up products
  const int kblocks = (a.d + kFp8Block - 1) / kFp8Block, fblocks = (a.F + kFp8Block - 1) / kFp8Block;
  const int wpt = sh.warps_per_tile;
  const int wi = warp & (wpt - 1), wt = warp / wpt;   // this warp's share of a tile, and its group of warps
  const int stride = (int)gridDim.x * (kWarps / wpt);
  int join = 0;   // the warps of a group count their tiles alike
  uint32_t parity = 0, joined = 0;
  float most[2 * NT] = {};
  for (int t0 = 0; t0 < a.T; t0 += per_group) {
    const int n = a.T - t0 < per_group ? a.T - t0 : per_group;
    if (a.groups > 1) {   // else the tokens are there, and all experts are of the group
      load_x(t0, n);
      scale_x(n, 0);
      const uint32_t in_group = ((1u << n) - 1u) << t0;
      if (warp == 0) {
        int m = 0;
        for (int u0 = 0; u0 < sh.used; u0 += 32) {
          const int u = u0 + lane;
          const bool has = u < sh.used && (sh.used_tokens[sh.list[u]] & in_group) != 0u;
          const uint32_t b = __ballot_sync(0xffffffffu, has);
          if (has) sh.group[m + __popc(b & ((1u << lane) - 1u))] = u;
          m += __popc(b);
        }
        if (lane == 0) sh.group_used = m;
      }
      __syncthreads();
      if (tid < kMaxTokens) sh.top[tid] = 0u;   // for the next group, behind load_x's barrier
    }
    const int tiles = sh.group_used * ftiles;

    uint32_t w0[kAhead][8], w1[kAhead][8];
    float f0[kAhead], f1[kAhead];
    const int first = (int)blockIdx.x * (kWarps / wpt) + wt;
    // the next load: tile and step
    int lt = first, ls = wi;
    const uint8_t *p0 = nullptr, *p1 = nullptr;
    const float *q0 = nullptr, *q1 = nullptr;
    auto aim = [&]() {
      if (lt >= tiles) return;
      const int gu = lt / ftiles, ft = lt - gu * ftiles;
      const int e = sh.list[sh.group[gu]];
      const int64_t at = ((int64_t)e * a.F + ft * 8 + g) * a.d * G::kBytes + c * 32 + ls * 128;
      p0 = a.w1 + at;
      p1 = a.w3 + at;
      if (FP8) {
        const int64_t sat = ((int64_t)e * fblocks + ft * 8 / kFp8Block) * kblocks + ls;
        q0 = a.s1 + sat;
        q1 = a.s3 + sat;
      }
    };
    auto load = [&](uint32_t (&x0)[8], uint32_t (&x1)[8], float& y0, float& y1) {
      if (lt >= tiles) return;
      if (ls * G::kStep + c * G::kPer < a.d) {
        ld_global_nc_v8(p0, x0);
        ld_global_nc_v8(p1, x1);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x0[i] = x1[i] = 0u;
      }
      if (FP8) {
        y0 = __ldg(q0);
        y1 = __ldg(q1);
        q0 += wpt;
        q1 += wpt;
      }
      p0 += wpt * 128;
      p1 += wpt * 128;
      ls += wpt;
      if (ls >= steps) {
        ls = wi;
        lt += stride;
        aim();
      }
    };
    aim();
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load(w0[i], w1[i], f0[i], f1[i]);

    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
    // this lane's place in the tokens' fragments
    const uint32_t step_bytes = (uint32_t)G::kPieces * n * 64;
    const uint8_t* xl = smem + lay.x + c * 16;
    int s = wi;
    bool ok = true;
    // The tokens of this lane's columns.  Up to 8 tokens: column t is token t, whether it chose the expert or not;
    // more: the expert's own one after the other, so that 8 or fewer of 16 take one product and not two.
    int mine_of[NT], columns = n;
    auto choose = [&](int tile) {
#pragma unroll
      for (int i = 0; i < NT; ++i) mine_of[i] = i * 8 + g;
      if (NT > 1 && tile < tiles) {
        const int u = tile / ftiles;   // (one group of tokens: sh.group is the identity)
        columns = __popc(sh.used_tokens[sh.list[u]]);
#pragma unroll
        for (int i = 0; i < NT; ++i)
          if (i * 8 + g < columns) mine_of[i] = sh.column[u][i * 8 + g];
      }
    };
    choose(first);
    for (int tile = first; tile < tiles && ok;) {
#pragma unroll
      for (int b = 0; b < kAhead; ++b) {
        if (tile >= tiles || !ok) break;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          if (i > 0 && columns <= 8 * i) continue;
          // two chains of dependent products
          float part[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
          const bool has = i * 8 + g < columns;
          const uint8_t* src = xl + s * step_bytes + mine_of[i] * 64;
#pragma unroll
          for (int p = 0; p < G::kPieces; ++p) {
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (has) v = *reinterpret_cast<const uint4*>(src + p * n * 64);
            mma_piece<FP8, M>(part[p & 1], w0[b], w1[b], p, v);
          }
          if (FP8) {
            acc[i][0] = fmaf(part[0][0] + part[1][0], f0[b], acc[i][0]);
            acc[i][1] = fmaf(part[0][1] + part[1][1], f0[b], acc[i][1]);
            acc[i][2] = fmaf(part[0][2] + part[1][2], f1[b], acc[i][2]);
            acc[i][3] = fmaf(part[0][3] + part[1][3], f1[b], acc[i][3]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] += part[0][j] + part[1][j];
          }
        }
        load(w0[b], w1[b], f0[b], f1[b]);
        s += wpt;
        if (s < steps) continue;
        // the tile's end: this warp's part
        s = wi;
        uint64_t *full = &sh.full[join][wt], *empty = &sh.empty[join][wt];
        ok = mbar_wait(empty, parity ^ 1u, &a.head->error, &sh.abort, kSite + 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        float* parts = red + join * kRedBuf + wt * wpt * kRedWarp;
        float* mine = parts + wi * kRedWarp;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          if (i * 8 + c * 2 < columns) {
            *reinterpret_cast<float2*>(mine + g * kRedRow + i * 8 + c * 2) = make_float2(acc[i][0], acc[i][1]);
            *reinterpret_cast<float2*>(mine + (g + 8) * kRedRow + i * 8 + c * 2) = make_float2(acc[i][2], acc[i][3]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(full);
        // ... and one of its warps, another each time, joins the parts
        if ((joined & (uint32_t)(wpt - 1)) == (uint32_t)wi) {
          ok = mbar_wait(full, parity, &a.head->error, &sh.abort, kSite + 2);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const int gu = tile / ftiles, ft = tile - gu * ftiles;
          const int u = sh.group[gu], e = sh.list[u];
          const uint32_t chosen = sh.used_tokens[e] >> t0;
          const int f = lane & 7;
#pragma unroll
          for (int i = 0; i < 2 * NT; ++i) {
            const int at = (lane >> 3) + 4 * i;   // column
            const int t = NT > 1 && at < columns ? sh.column[u][at] : at;
            if (at < columns && ((chosen >> t) & 1u)) {
              const float* r = parts + f * kRedRow + at;
              float gate = 0.0f, up = 0.0f;
#pragma unroll 4
              for (int w = 0; w < wpt; ++w) {
                gate += r[w * kRedWarp];
                up += r[w * kRedWarp + 8 * kRedRow];
              }
              gate *= sh.unscale[t];
              up *= sh.unscale[t];
              const float h = gate / (1.0f + expf(-gate)) * up * share[e * a.T + t0 + t];
              a.h[((int64_t)u * a.T + t0 + t) * a.F + ft * 8 + f] = h;
              if (NT > 1) {   // a column is another token with every expert
                if (fabsf(h) < kInf && __float_as_uint(fabsf(h)) > sh.htop[t]) atomicMax(&sh.htop[t], __float_as_uint(fabsf(h)));
              } else if (fabsf(h) < kInf) {
                most[i] = fmaxf(most[i], fabsf(h));
              }
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(empty);
        }
        ++joined;
        if (++join == kJoins) {
          join = 0;
          parity ^= 1u;
        }
        tile += stride;
        if (NT > 1) choose(tile);
      }
    }
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      const int t = (lane >> 3) + 4 * i;
      if (t < n && most[i] > 0.0f) atomicMax(&sh.htop[t0 + t], __float_as_uint(most[i]));
      most[i] = 0.0f;
    }
    __syncthreads();
  }
  if (tid < a.T) a.tops[(int64_t)blockIdx.x * a.T + tid] = sh.htop[tid];
  if (blockIdx.x == 0) {
    for (int i = tid; i < sh.used; i += kThreads) {
      a.head->expert[i] = sh.list[i];
      a.head->tokens[i] = sh.used_tokens[sh.list[i]];
    }
    if (tid == 0) a.head->used = sh.used;
    for (int i = tid; i < (a.d + kRowBlock - 1) / kRowBlock; i += kThreads) a.counters[i] = 0u;
  }
}

// ---------------------------------------------------------------------------------------
// second kernel
// ---------------------------------------------------------------------------------------
// The terms of a token's hidden values are neighbouring columns.  MODE 0: up to 4 tokens, in every expert's MMAs, whose
// sums stay in registers for the whole slice.  MODE 1, 2 (up to 8, 16 tokens): of each expert the tokens that chose it, one
// behind the other in as many MMAs as they fill, whose sums go to the tokens' own in shared memory at the expert's end (with
// all tokens in every expert's columns, 16 E4M3 tokens through 8 experts of 4096 x 14336 took this kernel 187 us, so 152).
// CHUNKS: a slice's hidden values do not fit shared memory at once.
template <bool FP8, typename X, int MODE, bool CHUNKS>
__global__ void __launch_bounds__(kThreads, 1) down_kernel(const FewArgs a) {
  using G = Geo<FP8>;
  using M = typename std::conditional<FP8, __half, X>::type;
  constexpr int kTerms = kTermsOf<FP8, X>;
  constexpr int kCols = kTerms == 2 ? 2 : 4, kPerMma = 8 / kCols;   // columns of a token (a fourth stays empty)
  constexpr int Q = (MODE == 2 ? 16 : (MODE == 1 ? 8 : 4)) / kPerMma;   // MMAs at most
  // Steps of weights in flight.  The sums of 9 to 16 tokens (16 or 32 a thread) leave registers for two; three terms for
  // three (with four, 4 tokens through 8 experts of 4096 x 14336 took 326 us, so 322; 8 tokens 554 and 492).
  constexpr int kAhead = MODE == 2 && (FP8 || kTerms == 3) ? 2 : (kTerms == 3 ? 3 : kAheadOf<FP8>);
  constexpr int kBurst = kAhead == 4 ? 2 : kAhead;
  static_assert(kChunkSteps % kAhead == 0, "a chunk starts at the first of the buffers in flight");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int expert[kMaxUsed];
  __shared__ uint32_t tokens[kMaxUsed];
  __shared__ uint32_t top[kMaxTokens];
  __shared__ uint8_t column[kMaxUsed][kMaxTokens];   // an expert's tokens, one after the other
  __shared__ int last;
  __shared__ uint32_t failed;   // a wait of the first kernel ran out: the output is NaN
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int T = a.T;
  if (tid < kMaxTokens) top[tid] = 0u;
  __syncthreads();
  wait_for_launcher();
  const int used = __ldcg(&a.head->used);
  if (tid == 0) failed = __ldcg(&a.head->error);
  for (int i = tid; i < a.E + a.S; i += kThreads) {   // (behind `used`: never looked at)
    expert[i] = __ldcg(&a.head->expert[i]);
    const uint32_t who = __ldcg(&a.head->tokens[i]);
    tokens[i] = who;
    uint32_t left = who & 0xffffu;
    for (int j = 0; left; ++j, left &= left - 1u) column[i][j] = (uint8_t)(__ffs(left) - 1);
  }
  for (int i = tid; i < a.grid1 * T; i += kThreads) {
    const uint32_t v = __ldcg(a.tops + i);
    if (v) atomicMax(&top[T == 1 ? 0 : i % T], v);
  }
  __syncthreads();
  const int fsteps = (a.F + G::kStep - 1) / G::kStep;
  const int total = used * fsteps;
  const int slices = a.split < total ? a.split : total;
  const int item = a.item0 + blockIdx.x, rb = item / a.split, slice = item % a.split;
  if (slice >= slices) return;
  const int begin = (int)((int64_t)total * slice / slices), end = (int)((int64_t)total * (slice + 1) / slices);
  const int row0 = rb * kRowBlock + warp * 16;
  const bool rows_ok = row0 < a.d;   // d is a multiple of 16
  const int fblocks = (a.F + kFp8Block - 1) / kFp8Block, dblocks = (a.d + kFp8Block - 1) / kFp8Block;

  // weights: the same pipeline as in the first kernel
  uint32_t w0[kAhead][8], w1[kAhead][8];
  float f[kAhead];
  int ls = begin, lu = begin / fsteps, lk = begin - lu * fsteps;
  const uint8_t* p0 = nullptr;
  const float* q0 = nullptr;
  const int64_t pitch = (int64_t)a.F * G::kBytes;
  auto aim = [&]() {
    if (ls >= end) return;
    const int e = expert[lu];
    p0 = a.w2 + ((int64_t)e * a.d + row0 + g) * pitch + c * 32 + lk * 128;
    if (FP8) q0 = a.s2 + ((int64_t)e * dblocks + row0 / kFp8Block) * fblocks + lk;
  };
  auto load = [&](uint32_t (&x0)[8], uint32_t (&x1)[8], float& y) {
    if (ls >= end) return;
    if (rows_ok && lk * G::kStep + c * G::kPer < a.F) {
      ld_global_nc_v8(p0, x0);
      ld_global_nc_v8(p0 + 8 * pitch, x1);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x0[i] = x1[i] = 0u;
    }
    if (FP8) y = rows_ok ? __ldg(q0++) : 0.0f;
    p0 += 128;
    ++ls;
    if (++lk == fsteps) {
      lk = 0;
      ++lu;
      aim();
    }
  };

  // Hidden values are staged as two or three 16-bit numbers (of values scaled to at most 2^15), in pieces of 8 of a
  // token; those of the next chunk beside this chunk's products.
  constexpr int kStepPieces = G::kStep / 8;
  const uint32_t step_bytes = (uint32_t)G::kPieces * T * kTerms * 64;   // [piece][token][term][lane of the quad]
  // Piece q of token t in a step of the contraction, zeros behind the last feature; false where the token did
  // not choose the expert: nobody looks there.
  auto fetch = [&](int step, int t, int q, float4& v0, float4& v1) {
    const int u = step / fsteps, kk = (step - u * fsteps) * G::kStep + q * 8;
    if (!((tokens[u] >> t) & 1u)) return false;
    v0 = v1 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (kk < a.F) {
      const float4* src = reinterpret_cast<const float4*>(a.h + ((int64_t)u * T + t) * a.F + kk);
      v0 = __ldcg(src);
      v1 = __ldcg(src + 1);
    }
    return true;
  };
  auto put_piece = [&](uint8_t* dst, float scale, const float4& v0, const float4& v1) {
    const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
    uint32_t term[kTerms][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x = v[2 * j] * scale, y = v[2 * j + 1] * scale;
#pragma unroll
      for (int i = 0; i < kTerms; ++i) {
        term[i][j] = narrow2<M>(x, y);
        const float2 r = widen2<M>(term[i][j]);
        // what is left, exactly (of an infinity or NaN nothing)
        x = fabsf(r.x) < kInf ? x - r.x : 0.0f;
        y = fabsf(r.y) < kInf ? y - r.y : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < kTerms; ++i)
      *reinterpret_cast<uint4*>(dst + i * 64) = make_uint4(term[i][0], term[i][1], term[i][2], term[i][3]);
  };
  {
    // the first chunk, its first pieces asked for before the weights; four pieces in flight a thread if there are many
    const int n = end - begin < a.chunk ? end - begin : a.chunk;
    const int pieces = n * T * kStepPieces;
    auto place = [&](int i) {
      const int q = i % kStepPieces, r = i / kStepPieces, t = T == 1 ? 0 : r % T, step = T == 1 ? r : r / T;
      return smem + step * step_bytes + ((uint32_t)(q % G::kPieces) * T + t) * (kTerms * 64) + q / G::kPieces * 16;
    };
    auto ask = [&](int i, float4& x, float4& y) {
      const int r = i / kStepPieces;
      return i < pieces && fetch(begin + (T == 1 ? r : r / T), T == 1 ? 0 : r % T, i % kStepPieces, x, y);
    };
    auto scale_of = [&](int i) { return pow2(range_exponent(top[T == 1 ? 0 : i / kStepPieces % T])); };
    float4 x, y;
    const bool have = ask(tid, x, y);
    aim();
#pragma unroll
    for (int j = 0; j < kAhead; ++j) load(w0[j], w1[j], f[j]);
    if (have) put_piece(place(tid), scale_of(tid), x, y);
#pragma unroll 1
    for (int i0 = tid + kThreads; i0 < pieces; i0 += 4 * kThreads) {
      float4 v[4][2];
      bool got[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) got[m] = ask(i0 + m * kThreads, v[m][0], v[m][1]);
#pragma unroll
      for (int m = 0; m < 4; ++m)
        if (got[m]) put_piece(place(i0 + m * kThreads), scale_of(i0 + m * kThreads), v[m][0], v[m][1]);
    }
  }
  __syncthreads();
  // One step of the next chunk at a time, its pieces (of the tokens that there are) over as many warps as they fill,
  // other warps each step.
  float4 v0, v1;
  uint32_t to = 0;
  float v_scale = 0.0f;
  bool pending = false;   // v0, v1 hold a piece
  int nu = 0, nk = 0;     // the next step to stage: expert, and step of it
  auto put_next = [&](uint8_t* stage) {
    if (pending) put_piece(stage + to, v_scale, v0, v1);
    pending = false;
  };
  auto fetch_next = [&](int step) {   // of the chunk
    const int first = ((warp + 5 * step) & (kWarps - 1)) * 32, piece = first + lane;
    const int pieces = __popc(tokens[nu]) * kStepPieces;
    if (first < pieces) {
      if (piece < pieces) {
        const int t = column[nu][piece / kStepPieces], q = piece % kStepPieces;
        pending = fetch(nu * fsteps + nk, t, q, v0, v1);
        to = step * step_bytes + ((uint32_t)(q % G::kPieces) * T + t) * (kTerms * 64) + q / G::kPieces * 16;
        v_scale = pow2(range_exponent(top[t]));
      }
      __syncwarp();
    }
    if (++nk == fsteps) {
      nk = 0;
      ++nu;
    }
  };

  float acc[Q][4];
#pragma unroll
  for (int i = 0; i < Q; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
  // MODE 1, 2: the tokens' sums of this warp's rows, [token][16 rows]
  float* sums = reinterpret_cast<float*>(smem + a.sums_at) + warp * 16 * T;
  if (MODE != 0) {
    for (int i = lane; i < 16 * T; i += 32) sums[i] = 0.0f;
    __syncwarp();
  }
  // this lane's columns: of MMA i a term of token i * kPerMma + g / kCols
  const uint32_t buf_bytes = step_bytes * a.chunk;
  int u = begin / fsteps, k = begin - u * fsteps, buf = 0, columns = 0;
  constexpr uint32_t kNone = 0xffffffffu;
  uint32_t from[Q];   // of the step's hidden values; kNone: no token
  // MODE 0: of the first MMA
  const uint32_t all_from = kTerms == 2 ? lane * 16 : (g / kCols * kTerms + g % kCols) * 64 + c * 16;
  auto choose = [&]() {   // of expert u
    if (MODE == 0) return;
    columns = __popc(tokens[u]);
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      const int at = i * kPerMma + g / kCols;
      from[i] = at < columns && g % kCols < kTerms ? (column[u][at] * kTerms + g % kCols) * 64 + c * 16 : kNone;
    }
  };
  // Sum of the terms of token i * kPerMma + c * 2 / kCols, rows g (r = 0) and g + 8 (r = 2), in the first of its lanes.
  auto token_sum = [&](int i, int r) {
    float v = acc[i][r] + acc[i][r + 1];
    if (kCols == 4) v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v;
  };
  const bool first_lane = kCols == 2 || (c & 1) == 0;
  auto deliver = [&]() {   // the sums of expert u's tokens
    if constexpr (MODE != 0) {
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        const int at = i * kPerMma + c * 2 / kCols;
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          const float v = token_sum(i, r);
          if (first_lane && at < columns) sums[column[u][at] * 16 + g + r * 4] += v;
          acc[i][r] = acc[i][r + 1] = 0.0f;
        }
      }
      __syncwarp();
    }
  };
  if (begin < end) choose();
  for (int at = begin; at < end; at += a.chunk, buf ^= 1) {
    const int n = end - at < a.chunk ? end - at : a.chunk;
    const int next = end - at - n < a.chunk ? end - at - n : a.chunk;   // steps of the next chunk
    uint8_t* other = smem + (buf ^ 1) * buf_bytes;
    if (CHUNKS) {
      nu = (at + n) / fsteps;
      nk = at + n - nu * fsteps;
    }
    for (int s0 = 0; s0 < n; s0 += kAhead) {
#pragma unroll
      for (int b = 0; b < kAhead; ++b) {
        const int s = s0 + b;
        if (s >= n) break;
        if (CHUNKS) {
          put_next(other);
          if (s < next) fetch_next(s);
        }
        const uint32_t mask = MODE == 0 ? tokens[u] : 0u;
        const uint8_t* src = smem + buf * buf_bytes + s * step_bytes;
        auto operand = [&](int i, int p) {
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (MODE == 0 ? (mask >> (i * kPerMma + g / kCols) & 1u) != 0u && g % kCols < kTerms : from[i] != kNone)
            v = *reinterpret_cast<const uint4*>(src + p * T * (kTerms * 64) +
                                                (MODE == 0 ? all_from + i * kPerMma * (kTerms * 64) : from[i]));
          return v;
        };
        auto add = [&](int i, const float (&v)[4]) {
          // (MODE 0: a token without the expert gets nothing, where zero times an infinite weight would be NaN)
          if (MODE == 0 && (mask >> (i * kPerMma + c * 2 / kCols) & 1u) == 0u) return;
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = FP8 ? fmaf(v[j], f[b], acc[i][j]) : acc[i][j] + v[j];
        };
        // Two MMAs at a time, a chain of dependent products each; one by itself: two chains.  (fp16, whose four steps in
        // flight leave no registers for that: one at a time.)
        constexpr bool kPairs = Q > 1 && (FP8 || kTerms == 3);
        constexpr int kNext = kPairs ? 1 : 0;
        const int have = MODE == 0 ? T : columns;
#pragma unroll
        for (int i = 0; i < Q; i += 1 + kNext) {
          if (i > 0 && have <= i * kPerMma) break;
          float part[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
          if (kPairs && have > (i + 1) * kPerMma) {
#pragma unroll
            for (int p = 0; p < G::kPieces; ++p) {
              const uint4 v0 = operand(i, p), v1 = operand(i + kNext, p);
              mma_piece<FP8, M>(part[0], w0[b], w1[b], p, v0);
              mma_piece<FP8, M>(part[1], w0[b], w1[b], p, v1);
            }
            add(i, part[0]);
            add(i + kNext, part[1]);
          } else {
#pragma unroll
            for (int p = 0; p < G::kPieces; ++p) mma_piece<FP8, M>(part[p & 1], w0[b], w1[b], p, operand(i, p));
#pragma unroll
            for (int j = 0; j < 4; ++j) part[0][j] += part[1][j];
            add(i, part[0]);
          }
        }
        if (b % kBurst == kBurst - 1) {
#pragma unroll
          for (int j = b - kBurst + 1; j <= b; ++j) load(w0[j], w1[j], f[j]);
        }
        if (++k == fsteps) {
          deliver();
          k = 0;
          if (++u < used) choose();
        }
      }
    }
    if (CHUNKS && next > 0) {
      put_next(other);
      __syncthreads();
    }
  }
  if (k > 0) deliver();

  // ---- the slices' sum
  auto put = [&](int t, int row, float v) {
    if constexpr (std::is_same<X, __half>::value)
      static_cast<__half*>(a.y)[(int64_t)t * a.d + row] = __float2half_rn(v);
    else
      static_cast<__nv_bfloat16*>(a.y)[(int64_t)t * a.d + row] = __float2bfloat16_rn(v);
  };
  auto give = [&](int t, int row, float v) {
    v = failed ? __uint_as_float(0x7fc00000u) : v * pow2(-range_exponent(top[t]));
    if (slices == 1)
      put(t, row, v);
    else
      a.part[((int64_t)slice * T + t) * a.d + row] = v;
  };
  if constexpr (MODE == 0) {
#pragma unroll
    for (int i = 0; i < Q; ++i)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const int t = i * kPerMma + c * 2 / kCols;
        const float v = token_sum(i, r);
        if (rows_ok && first_lane && t < T) give(t, row0 + g + r * 4, v);
      }
  } else if (rows_ok) {
    for (int i = lane; i < 16 * T; i += 32) give(i >> 4, row0 + (i & 15), sums[i]);
  }
  if (slices == 1) return;
  __syncthreads();   // all parts are written before thread 0's release
  if (tid == 0) {
    uint32_t before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], %2;" : "=r"(before) : "l"(a.counters + rb), "r"(1u) : "memory");
    last = before == (uint32_t)slices - 1u;
  }
  __syncthreads();
  if (!last) return;
  // four rows a thread, six slices' loads at a time, added in order
  for (int i = tid; i < T * kRowBlock / 4; i += kThreads) {
    const int t = i / (kRowBlock / 4), row = rb * kRowBlock + i % (kRowBlock / 4) * 4;
    if (row >= a.d) continue;
    const float* src = a.part + (int64_t)t * a.d + row;
    const int64_t step = (int64_t)T * a.d;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (int s0 = 0; s0 < slices; s0 += 6) {
      float4 p[6];
#pragma unroll
      for (int j = 0; j < 6; ++j)
        p[j] = s0 + j < slices ? __ldcg(reinterpret_cast<const float4*>(src + (s0 + j) * step)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < 6; ++j) {
        v[0] += p[j].x;
        v[1] += p[j].y;
        v[2] += p[j].z;
        v[3] += p[j].w;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) put(t, row + j, v[j]);
  }
}

// ---------------------------------------------------------------------------------------
struct FewWorkspace {
  size_t head, counters, tops, h, part, total;
};
FewWorkspace few_workspace(int T, int d, int F, int E, int k, int S) {
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  const int used = (E < T * k ? E : T * k) + S;
  const int blocks = (d + kRowBlock - 1) / kRowBlock;
  const int split = kSplitCtas / blocks > 1 ? kSplitCtas / blocks : 1;
  FewWorkspace w;
  w.head = 0;
  w.counters = up(sizeof(Header));
  w.tops = w.counters + up((size_t)blocks * 4);
  w.h = w.tops + up((size_t)kMaxCtas * T * 4);
  w.part = w.h + up((size_t)used * T * F * 4);
  w.total = w.part + up((size_t)split * T * d * 4);
  return w;
}

template <bool FP8, typename X>
int launch(FewArgs a, int items, int ctas, bool limited, uint32_t smem1, cudaStream_t stream) {
  const uint32_t step_bytes = (uint32_t)Geo<FP8>::kStep * a.T * 2 * kTermsOf<FP8, X>;
  const int used = (a.E < a.T * a.k ? a.E : a.T * a.k) + a.S;
  const int64_t most = ((int64_t)used * ((a.F + Geo<FP8>::kStep - 1) / Geo<FP8>::kStep) + a.split - 1) / a.split + 1;
  const bool whole = most * step_bytes <= (kTermsOf<FP8, X> == 3 ? kWholeBytes3 : kWholeBytes);
  const int fit = (int)(kStageBytes / step_bytes) / kChunkSteps * kChunkSteps;
  a.chunk = whole ? (int)most : (fit > kChunkSteps ? fit : kChunkSteps);
  a.sums_at = (whole ? 1 : 2) * a.chunk * step_bytes;
  const uint32_t smem2 = a.sums_at + (a.T > 4 ? kWarps * 16 * a.T * 4 : 0);
  const bool two = a.T > 8 && a.groups == 1;
  auto k1 = two ? gate_up_kernel<FP8, X, 2> : gate_up_kernel<FP8, X, 1>;
  auto k2 = whole ? (a.T <= 4   ? down_kernel<FP8, X, 0, false>
                     : a.T <= 8 ? down_kernel<FP8, X, 1, false>
                                : down_kernel<FP8, X, 2, false>)
                  : (a.T <= 4   ? down_kernel<FP8, X, 0, true>
                     : a.T <= 8 ? down_kernel<FP8, X, 1, true>
                                : down_kernel<FP8, X, 2, true>);
  int st = set_max_dynamic_smem(reinterpret_cast<const void*>(k1), smem1);
  if (st != LMOE_OK) return st;
  st = set_max_dynamic_smem(reinterpret_cast<const void*>(k2), smem2);
  if (st != LMOE_OK) return st;
  k1<<<a.grid1, kThreads, smem1, stream>>>(a);
  LMOE_CUDA_TRY(cudaGetLastError());
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = smem2;
  config.stream = stream;
  config.attrs = &early;
  // One launch (items <= SMs).  Under a limit of CTAs several, each behind the other and the first behind the first kernel,
  // whose CTAs hold the limit's SMs: the slices, and with them the order of the sums, stay the same.
  config.numAttrs = limited ? 0 : 1;
  for (a.item0 = 0; a.item0 < items; a.item0 += ctas) {
    config.gridDim = dim3((unsigned)(items - a.item0 < ctas ? items - a.item0 : ctas));
    LMOE_CUDA_TRY(cudaLaunchKernelEx(&config, k2, a));
    config.numAttrs = 0;
  }
  return LMOE_OK;
}

bool few_sizes(int64_t T, int d, int F, int E, int k, int S) {
  return T >= 0 && T <= kMaxTokens && d >= 64 && d % 64 == 0 && d <= 16384 && F >= 32 && F % 32 == 0 && F <= 65536 &&
         E >= 1 && E <= kMaxExperts && k >= 1 && k <= kMaxTopK && k <= E && S >= 0 && S <= kMaxShared;
}

}  // namespace
}  // namespace lmoe

using namespace lmoe;

extern "C" size_t lmoe_few_tokens_workspace_bytes(int64_t num_tokens, int hidden_size, int ffn_size, int num_experts,
                                                  int top_k, int num_shared) {
  if (!few_sizes(num_tokens, hidden_size, ffn_size, num_experts, top_k, num_shared)) return 0;
  return few_workspace((int)num_tokens, hidden_size, ffn_size, num_experts, top_k, num_shared).total;
}

extern "C" int lmoe_moe_layer_few_tokens(const void* x, int dtype, int64_t num_tokens, int hidden_size,
                                         const void* gate_weight, const float* gate_bias, int num_experts, int top_k,
                                         int num_shared, const void* w1, const void* w3, const void* w2,
                                         const float* w1_scales, const float* w3_scales, const float* w2_scales,
                                         int ffn_size, void* y, int32_t* ids, float* weights, void* workspace,
                                         size_t workspace_bytes, lmoe_stream_t stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  LMOE_ARG_CHECK(dtype == LMOE_DTYPE_BF16 || dtype == LMOE_DTYPE_F16);
  LMOE_ARG_CHECK(few_sizes(num_tokens, hidden_size, ffn_size, num_experts, top_k, num_shared));
  const bool fp8 = w1_scales != nullptr;
  LMOE_ARG_CHECK((w3_scales != nullptr) == fp8 && (w2_scales != nullptr) == fp8);
  if (num_tokens == 0) return LMOE_OK;
  LMOE_ARG_CHECK(x && gate_weight && w1 && w3 && w2 && y && ids && weights);
  LMOE_ARG_CHECK(aligned16(x) && aligned16(gate_weight) && aligned32(w1) && aligned32(w3) && aligned32(w2));
  LMOE_ARG_CHECK(((reinterpret_cast<uintptr_t>(gate_bias) | reinterpret_cast<uintptr_t>(w1_scales) |
                   reinterpret_cast<uintptr_t>(w3_scales) | reinterpret_cast<uintptr_t>(w2_scales) |
                   reinterpret_cast<uintptr_t>(ids) | reinterpret_cast<uintptr_t>(weights)) & 3) == 0);
  LMOE_ARG_CHECK((reinterpret_cast<uintptr_t>(y) & 1) == 0);
  const int T = (int)num_tokens;
  const FewWorkspace ws = few_workspace(T, hidden_size, ffn_size, num_experts, top_k, num_shared);
  if (!workspace || workspace_bytes < ws.total || !aligned16(workspace)) return LMOE_ERR_WORKSPACE;
  DeviceInfo dev;
  int st = get_device_info(&dev);
  if (st != LMOE_OK) return st;
  if (dev.cc_major != 10) return LMOE_ERR_DEVICE;
  FewArgs a = {};
  a.x = x;
  a.gate = gate_weight;
  a.bias = gate_bias;
  a.w1 = static_cast<const uint8_t*>(w1);
  a.w3 = static_cast<const uint8_t*>(w3);
  a.w2 = static_cast<const uint8_t*>(w2);
  a.s1 = w1_scales;
  a.s3 = w3_scales;
  a.s2 = w2_scales;
  a.T = T;
  a.d = hidden_size;
  a.F = ffn_size;
  a.E = num_experts;
  a.k = top_k;
  a.S = num_shared;
  a.y = y;
  a.ids = ids;
  a.weights = weights;
  uint8_t* base = static_cast<uint8_t*>(workspace);
  a.head = reinterpret_cast<Header*>(base + ws.head);
  a.counters = reinterpret_cast<uint32_t*>(base + ws.counters);
  a.tops = reinterpret_cast<uint32_t*>(base + ws.tops);
  a.h = reinterpret_cast<float*>(base + ws.h);
  a.part = reinterpret_cast<float*>(base + ws.part);
  // All tokens of a large layer may not fit shared memory: then eight at a time, each group reading
  // its experts' gate and up weights.
  const uint32_t limit = (uint32_t)dev.max_smem_optin - (uint32_t)sizeof(FewShared) - 1024;
  const int step = fp8 ? 128 : 64;
  a.groups = 1;
  uint32_t smem1 = few_layout(a.d, step, T, T, a.E + a.S).total;
  if (smem1 > limit) {
    a.groups = (T + 7) / 8;
    smem1 = few_layout(a.d, step, 8, T, a.E + a.S).total;
    if (smem1 > limit || a.groups < 2) return LMOE_ERR_UNSUPPORTED;
  }
  const int blocks = (a.d + kRowBlock - 1) / kRowBlock;
  a.split = kSplitCtas / blocks > 1 ? kSplitCtas / blocks : 1;
  const int ctas = gemm_grid(dev) < kMaxCtas ? gemm_grid(dev) : kMaxCtas;
  a.grid1 = ctas < 2 ? 2 : ctas & ~1;   // whole pairs
  const int items = blocks * a.split;
  const bool limited = gemm_grid(dev) < dev.num_sms;
  if (dtype == LMOE_DTYPE_BF16)
    return fp8 ? launch<true, __nv_bfloat16>(a, items, ctas, limited, smem1, stream)
               : launch<false, __nv_bfloat16>(a, items, ctas, limited, smem1, stream);
  return fp8 ? launch<true, __half>(a, items, ctas, limited, smem1, stream)
             : launch<false, __half>(a, items, ctas, limited, smem1, stream);
}
