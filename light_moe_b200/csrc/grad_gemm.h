// grad_gemm.h -- internal interface of the grouped product's gradients and the product of any row
// length (grad_gemm.cu for 16-bit operands; for fp32 grad_split.cu on tensor cores and grad_f32.cu
// on CUDA cores).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace lmoe {

enum GradForm : int {
  kGradInput = 0,     // dx[r, k] from dy and w
  kGradWeight = 1,    // dw[e, n, k] from dy and x
  kGradProduct = 2,   // y[r, n] from x and w: N below is the contraction (x's columns), K y's columns
};

struct GradProblem {
  int form = kGradInput;
  int dtype = 0;              // operands
  int out_dtype = 0;
  int64_t total_rows = 0;
  int N = 0, K = 0;
  int num_experts = 0;
  const void* dy = nullptr;      // [total_rows, N] (the product: x)
  const void* other = nullptr;   // w [num_experts, N, K], x [total_rows, K], or w [num_experts, K, N]
  const void* offsets = nullptr;
  int offsets_i64 = 0;
  void* out = nullptr;
  void* workspace = nullptr;     // copies of operands: padded rows, or planes of fp32; sums of ranges
  size_t workspace_bytes = 0;
  uint32_t* err = nullptr;
};

size_t grad_gemm_workspace(const GradProblem& p);
size_t grad_gemm_needs(const GradProblem& p);   // without it a call is refused
int run_grad_gemm(const GradProblem& p, cudaStream_t stream);
// Whether fp32 operands go to the tensor cores as three bf16 planes each.
bool grad_splits(const GradProblem& p);
size_t grad_split_workspace(const GradProblem& p);
int run_grad_split(const GradProblem& p, cudaStream_t stream);
int run_grad_f32(const GradProblem& p, cudaStream_t stream);

}  // namespace lmoe
