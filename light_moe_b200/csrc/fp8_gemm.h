// fp8_gemm.h -- internal interface of the grouped product of 8-bit operands (fp8_gemm.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace lmoe {

struct Fp8Problem {
  // rows: codes [total_rows, K] and scales [K blocks][xs_pitch elements]
  const uint8_t* xq = nullptr;
  const float* xs = nullptr;
  int64_t xs_pitch = 0;
  int64_t total_rows = 0;
  int K = 0;
  // weights: codes [num_experts, N, K] and scales [num_experts, N blocks, K blocks]; with an up
  // matrix the first is the gate and the output silu(gate) * up
  const uint8_t* wq = nullptr;
  const float* ws = nullptr;
  const uint8_t* wq_up = nullptr;
  const float* ws_up = nullptr;
  int N = 0;
  const void* offsets = nullptr;
  int offsets_i64 = 0;
  int num_experts = 0;
  int out_dtype = 0;
  void* out = nullptr;               // [total_rows, N]
  uint32_t* err = nullptr;
};

int run_fp8_gemm(const Fp8Problem& p, cudaStream_t stream);

}  // namespace lmoe
