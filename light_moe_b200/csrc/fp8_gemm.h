// fp8_gemm.h -- internal interface of the grouped product of 8-bit operands (fp8_gemm.cu, fp8_decode.cu).
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

int run_fp8_gemm(const Fp8Problem& p, cudaStream_t stream);     // many rows per expert
int run_fp8_decode(const Fp8Problem& p, cudaStream_t stream);   // few
constexpr int kFp8DecodeRows = 64;   // rows of a tile of run_fp8_decode

// Instruction descriptor of kind::f8f6f4: E4M3 operands, K-major, fp32 sums, M = 256, N = n.
__host__ __device__ constexpr uint32_t idesc_fp8(uint32_t n) {
  return (1u << 4) | ((n >> 3) << 17) | ((256u >> 4) << 24);
}
#ifdef __CUDACC__
__device__ __forceinline__ void mma_fp8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
#endif

}  // namespace lmoe
