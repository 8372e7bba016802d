// fp4_gemm.h -- internal interface of the grouped product of 4-bit operands (fp4_gemm.cu,
// fp4_decode.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace lmoe {

struct Fp4Problem {
  // rows: codes [total_rows, K / 2] and scales [total_rows, xs_pitch bytes]
  const uint8_t* xq = nullptr;
  const uint8_t* xs = nullptr;
  int64_t xs_pitch = 0;
  int64_t total_rows = 0;
  int K = 0;
  // weights: codes [num_experts, N, K / 2] and scales [num_experts, N, ws_pitch bytes]; with an up
  // matrix the first is the gate and the output silu(gate) * up
  const uint8_t* wq = nullptr;
  const uint8_t* ws = nullptr;
  const uint8_t* wq_up = nullptr;
  const uint8_t* ws_up = nullptr;
  int64_t ws_pitch = 0;
  int N = 0;
  int format = 0;
  const void* offsets = nullptr;
  int offsets_i64 = 0;
  int num_experts = 0;
  const float* alpha = nullptr;      // factor per expert (the product of the tensor scales)
  const float* alpha_up = nullptr;
  int out_dtype = 0;
  void* out = nullptr;               // [total_rows, N]
  uint32_t* err = nullptr;
};

int run_fp4_gemm(const Fp4Problem& p, cudaStream_t stream);     // many rows per expert
int run_fp4_decode(const Fp4Problem& p, cudaStream_t stream);   // few
constexpr int kFp4DecodeRows = 64;   // rows of a tile of run_fp4_decode

}  // namespace lmoe
