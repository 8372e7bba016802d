// bindings.cpp -- the `_C` operator module: light-moe's operator surface
// (csrc/bindings.cpp:28-49 of the reference: grouped_gemm, fused_gate_topk,
// fused_gate_topk_permute, same argument names and return types) plus the new W4A16 and
// MoE-layer ops, all implemented by calling the C ABI in include/lmoe_b200.h.
//
// Host-side duties only: argument checks (TORCH_CHECK -> RuntimeError, like the
// reference's fused_moe_ops.cu:150-151 / grouped_gemm.cu:17-18), output allocation through
// the PyTorch caching allocator, the device guard, and launching on the *current* CUDA
// stream (the reference launches its kernel on the legacy default stream).
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "lmoe_b200.h"

namespace {

void check_status(int st, const char* what) {
  TORCH_CHECK(st == LMOE_OK, what, " failed: ", lmoe_status_string(st), " (status ", st, ")");
}

lmoe_stream_t cur_stream() { return reinterpret_cast<lmoe_stream_t>(at::cuda::getCurrentCUDAStream().stream()); }

torch::Tensor as_bf16_contig(const torch::Tensor& t) {
  return t.scalar_type() == torch::kBFloat16 ? t.contiguous() : t.to(torch::kBFloat16).contiguous();
}

// The operand as one of the library's element types: bf16, fp16 and fp32 pass unchanged;
// any other floating type becomes fp32, the type the reference converts every operand to
// (csrc/fused_moe_ops.cu:158-159).
torch::Tensor as_kernel_type(const torch::Tensor& t) {
  const auto st = t.scalar_type();
  if (st == torch::kBFloat16 || st == torch::kFloat16 || st == torch::kFloat32) return t.contiguous();
  return t.to(torch::kFloat32).contiguous();
}

int dtype_code(const torch::Tensor& t) {
  switch (t.scalar_type()) {
    case torch::kBFloat16: return LMOE_DTYPE_BF16;
    case torch::kFloat16: return LMOE_DTYPE_F16;
    case torch::kFloat32: return LMOE_DTYPE_F32;
    default: TORCH_CHECK(false, "unsupported dtype ", t.scalar_type());
  }
  return -1;
}

void check_cuda(const torch::Tensor& t, const char* name) { TORCH_CHECK(t.is_cuda(), name, " must be CUDA"); }

torch::Tensor workspace(int64_t bytes, const torch::Tensor& like) {
  return torch::empty({bytes > 0 ? bytes : 1}, like.options().dtype(torch::kUInt8));
}

// Sizes that the kernels count in 32 bits.
void check_sizes(int64_t rows, int64_t n, int64_t k, int64_t num_experts) {
  TORCH_CHECK(rows <= INT32_MAX && n <= INT32_MAX && k <= INT32_MAX && num_experts <= INT32_MAX,
              "sizes must fit 32 bits");
}

// Row-contiguous and 16-byte aligned (a view may start anywhere).
torch::Tensor contig16(const torch::Tensor& t) {
  auto c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}

struct Routed {
  torch::Tensor ids, weights, counts, offsets, sorted_idx, positions, logits, probs;
};

Routed route(const torch::Tensor& hidden_states, const torch::Tensor& gate_weight,
             const std::optional<torch::Tensor>& bias, int64_t top_k, bool perm, bool want_logits,
             bool want_probs = false) {
  check_cuda(hidden_states, "hidden_states");
  check_cuda(gate_weight, "gate_weight");
  TORCH_CHECK(hidden_states.dim() == 2 && gate_weight.dim() == 2, "hidden_states [T,d] and gate_weight [E,d]");
  TORCH_CHECK(hidden_states.size(1) == gate_weight.size(1), "hidden size mismatch");
  const c10::cuda::OptionalCUDAGuard guard(hidden_states.device());
  auto x = as_kernel_type(hidden_states);
  auto w = as_kernel_type(gate_weight);
  const int64_t T = x.size(0);
  const int64_t d = x.size(1);
  const int64_t E = w.size(0);
  torch::Tensor b;
  if (bias.has_value() && bias->defined()) {
    check_cuda(*bias, "bias");
    b = bias->to(torch::kFloat32).contiguous();
    TORCH_CHECK(b.numel() == E, "bias must have num_experts elements");
  }
  auto i32 = x.options().dtype(torch::kInt32);
  Routed r;
  r.ids = torch::empty({T, top_k}, i32);
  r.weights = torch::empty({T, top_k}, x.options().dtype(torch::kFloat32));
  if (perm) {
    r.counts = torch::empty({E}, i32);
    r.offsets = torch::empty({E + 1}, i32);
    r.sorted_idx = torch::empty({T * top_k}, i32);
    r.positions = torch::empty({T * top_k}, i32);
  }
  if (want_logits) r.logits = torch::empty({T, E}, x.options().dtype(torch::kFloat32));
  if (want_probs) r.probs = torch::empty({T, E}, x.options().dtype(torch::kFloat32));
  const int xdt = dtype_code(x), wdt = dtype_code(w);
  auto ws = workspace((int64_t)lmoe_router_workspace_bytes_typed(T, (int)E, xdt, wdt), x);
  int st = lmoe_fused_gate_topk_typed(x.data_ptr(), xdt, w.data_ptr(), wdt, b.defined() ? b.data_ptr<float>() : nullptr,
                                T, (int)d,
                                (int)E, (int)top_k, r.ids.data_ptr<int32_t>(), r.weights.data_ptr<float>(), nullptr,
                                perm ? r.counts.data_ptr<int32_t>() : nullptr,
                                perm ? r.offsets.data_ptr<int32_t>() : nullptr,
                                perm ? r.sorted_idx.data_ptr<int32_t>() : nullptr,
                                perm ? r.positions.data_ptr<int32_t>() : nullptr,
                                want_logits ? r.logits.data_ptr<float>() : nullptr,
                                want_probs ? r.probs.data_ptr<float>() : nullptr, ws.data_ptr(), ws.numel(),
                                cur_stream());
  check_status(st, "fused_gate_topk");
  return r;
}

// ---------------------------------------------------------------- reference surface

// light_moe._C.fused_gate_topk (csrc/bindings.cpp:38-42 of the reference)
std::tuple<torch::Tensor, torch::Tensor> fused_gate_topk(torch::Tensor hidden_states, torch::Tensor gate_weight,
                                                         int64_t top_k) {
  Routed r = route(hidden_states, gate_weight, std::nullopt, top_k, false, false);
  return {r.ids, r.weights.to(hidden_states.scalar_type())};
}

// light_moe._C.fused_gate_topk_permute (csrc/bindings.cpp:44-48 of the reference)
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> fused_gate_topk_permute(
    torch::Tensor hidden_states, torch::Tensor gate_weight, int64_t top_k) {
  Routed r = route(hidden_states, gate_weight, std::nullopt, top_k, true, false);
  const c10::cuda::OptionalCUDAGuard guard(hidden_states.device());
  // the permuted rows are the caller's rows, copied unchanged in their own dtype
  auto x = hidden_states.contiguous();
  const int64_t T = x.size(0);
  const int64_t d = x.size(1);
  auto permuted = torch::empty({T * top_k, d}, x.options());
  const int esize = (int)x.element_size();
  int st = LMOE_OK;
  if ((esize == 2 || esize == 4) && (d * esize) % 16 == 0) {
    st = lmoe_permute_rows(x.data_ptr(), esize, r.sorted_idx.data_ptr<int32_t>(), T * top_k, (int)d, (int)top_k,
                           permuted.data_ptr(), cur_stream());
  } else {
    // other element sizes or row lengths: the same gather through ATen
    permuted = x.index_select(0, r.sorted_idx.to(torch::kInt64).floor_divide(top_k));
  }
  check_status(st, "fused_gate_topk_permute");
  return {permuted, r.ids, r.weights.to(hidden_states.scalar_type()),
          r.offsets.to(torch::kInt64), r.sorted_idx.to(torch::kInt64)};
}

// light_moe._C.grouped_gemm (csrc/bindings.cpp:32-36 of the reference)
torch::Tensor grouped_gemm(torch::Tensor input, torch::Tensor weights, torch::Tensor expert_offsets,
                           int64_t num_experts) {
  check_cuda(input, "input");
  check_cuda(weights, "weights");
  check_cuda(expert_offsets, "expert_offsets");
  TORCH_CHECK(input.dim() == 2 && weights.dim() == 3, "input [T,K], weights [E,N,K]");
  TORCH_CHECK(weights.size(0) >= num_experts && weights.size(2) == input.size(1), "shape mismatch");
  TORCH_CHECK(expert_offsets.numel() >= num_experts + 1, "expert_offsets must have num_experts + 1 entries");
  check_sizes(input.size(0), weights.size(1), input.size(1), num_experts);
  const c10::cuda::OptionalCUDAGuard guard(input.device());
  // computed in the input dtype (bf16 / fp16 on tensor cores, fp32 on CUDA cores), like the
  // reference's per-expert mm_out (csrc/grouped_gemm.cu:24-40); the weights follow the input
  auto x = contig16(as_kernel_type(input));
  auto w = contig16(weights.scalar_type() == x.scalar_type() ? weights : weights.to(x.scalar_type()));
  auto off = expert_offsets.contiguous();
  TORCH_CHECK(off.scalar_type() == torch::kInt64 || off.scalar_type() == torch::kInt32, "offsets int64/int32");
  const int64_t T = x.size(0), K = x.size(1), N = w.size(1);
  auto out = torch::empty({T, N}, x.options());
  if (T == 0 && num_experts >= 1) return out.to(input.scalar_type());   // no rows, nothing to launch
  // row lengths that the kernels above do not take
  if (K > 0 && N > 0 && (x.scalar_type() == torch::kFloat32 ? K % 4 != 0 : K % 128 != 0)) {
    const int dt = dtype_code(x);
    auto ws = workspace((int64_t)lmoe_grouped_gemm_grad_workspace_bytes(2, dt, T, (int)N, (int)K, (int)num_experts), x);
    check_status(lmoe_grouped_gemm_any(x.data_ptr(), dt, T, (int)K, w.data_ptr(), (int)N, off.data_ptr(),
                                       off.scalar_type() == torch::kInt64 ? 1 : 0, (int)num_experts, out.data_ptr(),
                                       ws.data_ptr(), ws.numel(), nullptr, cur_stream()),
                 "grouped_gemm");
    return out.to(input.scalar_type());
  }
  auto ws = workspace((int64_t)lmoe_gemm_workspace_bytes(), x);
  int st = lmoe_grouped_gemm(x.data_ptr(), dtype_code(x), T, (int)K, w.data_ptr(), (int)N, off.data_ptr(),
                             off.scalar_type() == torch::kInt64 ? 1 : 0, (int)num_experts, 1, out.data_ptr(),
                             ws.data_ptr(), ws.numel(), cur_stream());
  check_status(st, "grouped_gemm");
  return out.to(input.scalar_type());
}

// ---------------------------------------------------------------- new ops

std::vector<torch::Tensor> fused_gate_topk_ex(torch::Tensor hidden_states, torch::Tensor gate_weight, int64_t top_k,
                                              std::optional<torch::Tensor> bias, bool return_logits,
                                              bool return_probs) {
  Routed r = route(hidden_states, gate_weight, bias, top_k, true, return_logits, return_probs);
  std::vector<torch::Tensor> out = {r.ids, r.weights, r.counts, r.offsets, r.sorted_idx, r.positions};
  if (return_logits) out.push_back(r.logits);
  if (return_probs) out.push_back(r.probs);
  return out;
}

std::tuple<torch::Tensor, torch::Tensor> quantize_w4(torch::Tensor w, int64_t group_size) {
  check_cuda(w, "w");
  TORCH_CHECK(w.dim() >= 2, "w must be [..., N, K]");
  const c10::cuda::OptionalCUDAGuard guard(w.device());
  const bool f32 = w.scalar_type() == torch::kFloat32;
  auto wc = f32 ? w.contiguous() : as_bf16_contig(w);
  const int64_t K = wc.size(-1);
  TORCH_CHECK(K % group_size == 0 && group_size % 2 == 0, "K must be divisible by an even group_size");
  const int64_t rows = wc.numel() / K;
  auto qshape = wc.sizes().vec();
  qshape.back() = K / 2;
  auto sshape = wc.sizes().vec();
  sshape.back() = K / group_size;
  auto q = torch::empty(qshape, wc.options().dtype(torch::kUInt8));
  auto s = torch::empty(sshape, wc.options().dtype(torch::kFloat16));
  int st = lmoe_quantize_w4(wc.data_ptr(), f32 ? 1 : 0, rows, (int)K, (int)group_size, q.data_ptr<uint8_t>(),
                            reinterpret_cast<uint16_t*>(s.data_ptr()), cur_stream());
  check_status(st, "quantize_w4");
  return {q, s};
}

torch::Tensor dequantize_w4(torch::Tensor qweight, torch::Tensor scales, int64_t group_size) {
  check_cuda(qweight, "qweight");
  check_cuda(scales, "scales");
  TORCH_CHECK(qweight.scalar_type() == torch::kUInt8 && scales.scalar_type() == torch::kFloat16, "uint8 / fp16");
  const c10::cuda::OptionalCUDAGuard guard(qweight.device());
  auto q = qweight.contiguous();
  auto s = scales.contiguous();
  const int64_t K = q.size(-1) * 2;
  const int64_t rows = q.numel() / (K / 2);
  TORCH_CHECK(s.numel() == rows * (K / group_size), "scales shape mismatch");
  auto shape = q.sizes().vec();
  shape.back() = K;
  auto out = torch::empty(shape, q.options().dtype(torch::kBFloat16));
  int st = lmoe_dequantize_w4(q.data_ptr<uint8_t>(), reinterpret_cast<const uint16_t*>(s.data_ptr()), rows, (int)K,
                              (int)group_size, out.data_ptr(), cur_stream());
  check_status(st, "dequantize_w4");
  return out;
}

torch::Tensor prepack_w4(torch::Tensor qweight, torch::Tensor scales, int64_t group_size,
                         std::optional<torch::Tensor> qweight_up, std::optional<torch::Tensor> scales_up) {
  check_cuda(qweight, "qweight");
  TORCH_CHECK(qweight.dim() == 3, "qweight must be [E, N, K/2]");
  const c10::cuda::OptionalCUDAGuard guard(qweight.device());
  auto q = qweight.contiguous();
  auto s = scales.contiguous();
  const bool paired = qweight_up.has_value() && qweight_up->defined();
  torch::Tensor qb, sb;
  if (paired) {
    qb = qweight_up->contiguous();
    sb = scales_up.value().contiguous();
    TORCH_CHECK(qb.sizes() == q.sizes() && sb.sizes() == s.sizes(), "gate and up shapes differ");
  }
  const int64_t E = q.size(0), N = q.size(1), K = q.size(2) * 2;
  size_t pb = 0;
  check_status(lmoe_w4_prepacked_bytes((int)E, (int)N, (int)K, (int)group_size, paired ? 1 : 0, &pb), "prepack_w4");
  auto packed = torch::empty({(int64_t)pb}, q.options());
  int st = lmoe_prepack_w4(q.data_ptr<uint8_t>(), reinterpret_cast<const uint16_t*>(s.data_ptr()),
                           paired ? qb.data_ptr<uint8_t>() : nullptr,
                           paired ? reinterpret_cast<const uint16_t*>(sb.data_ptr()) : nullptr, (int)E, (int)N,
                           (int)K, (int)group_size, packed.data_ptr<uint8_t>(), cur_stream());
  check_status(st, "prepack_w4");
  return packed;
}

torch::Tensor w4a16_grouped_gemm(torch::Tensor input, torch::Tensor packed, torch::Tensor expert_offsets, int64_t num_experts, int64_t N, int64_t group_size,
                                 int64_t epilogue, std::optional<torch::Tensor> dest_rows,
                                 std::optional<torch::Tensor> row_scale, int64_t out_rows,
                                 int64_t max_rows_per_expert, std::optional<torch::Tensor> segment_expert) {
  check_cuda(input, "input");
  check_cuda(packed, "packed");
  const c10::cuda::OptionalCUDAGuard guard(input.device());
  auto x = as_bf16_contig(input);
  auto off = expert_offsets.contiguous();
  const int64_t T = x.size(0), K = x.size(1);
  const int64_t ncols = epilogue == 1 ? N / 2 : N;
  const int64_t rows_out = out_rows > 0 ? out_rows : T;
  auto out = epilogue == 2 ? torch::zeros({rows_out, ncols}, x.options()) : torch::empty({rows_out, ncols}, x.options());
  torch::Tensor dr, rs;
  if (dest_rows.has_value() && dest_rows->defined()) dr = dest_rows->to(torch::kInt32).contiguous();
  if (row_scale.has_value() && row_scale->defined()) rs = row_scale->to(torch::kFloat32).contiguous();
  torch::Tensor se;
  if (segment_expert.has_value() && segment_expert->defined()) se = segment_expert->to(torch::kInt32).contiguous();
  // weight matrices held by `packed` (each N x K in the prepacked layout)
  size_t per = 0;
  check_status(lmoe_w4_prepacked_bytes(1, (int)N, (int)K, (int)group_size, 0, &per), "w4a16_grouped_gemm");
  TORCH_CHECK(per > 0 && packed.numel() % (int64_t)per == 0, "packed size is not a whole number of matrices");
  const int num_w = (int)(packed.numel() / (int64_t)per);
  auto ws = workspace((int64_t)lmoe_gemm_workspace_bytes(), x);
  int st = lmoe_w4a16_grouped_gemm(
      x.data_ptr(), T, (int)K, packed.data_ptr<uint8_t>(), (int)N, (int)group_size, off.data_ptr(), off.scalar_type() == torch::kInt64 ? 1 : 0, (int)num_experts,
      se.defined() ? se.data_ptr<int32_t>() : nullptr, num_w, (int)epilogue, dr.defined() ? dr.data_ptr<int32_t>() : nullptr, rs.defined() ? rs.data_ptr<float>() : nullptr,
      max_rows_per_expert, out.data_ptr(), ncols, ws.data_ptr(), ws.numel(), cur_stream());
  check_status(st, "w4a16_grouped_gemm");
  return out;
}

torch::Tensor combine_rows(torch::Tensor rows, torch::Tensor positions, torch::Tensor weights, int64_t num_tokens,
                           int64_t top_k, std::optional<torch::Tensor> extra_rows, int64_t num_extra) {
  check_cuda(rows, "rows");
  const c10::cuda::OptionalCUDAGuard guard(rows.device());
  auto r = as_bf16_contig(rows);
  auto p = positions.to(torch::kInt32).contiguous();
  auto w = weights.to(torch::kFloat32).contiguous();
  const int64_t d = r.size(1);
  torch::Tensor ex;
  if (extra_rows.has_value() && extra_rows->defined()) ex = as_bf16_contig(*extra_rows);
  auto y = torch::empty({num_tokens, d}, r.options());
  int st = lmoe_combine_rows(r.data_ptr(), p.data_ptr<int32_t>(), w.data_ptr<float>(), num_tokens, (int)top_k, (int)d,
                             ex.defined() ? ex.data_ptr() : nullptr, ex.defined() ? (int)num_extra : 0, y.data_ptr(),
                             cur_stream());
  check_status(st, "combine_rows");
  return y;
}

std::vector<torch::Tensor> moe_layer_w4a16(torch::Tensor x, torch::Tensor gate_weight, torch::Tensor w13_packed,
                                           torch::Tensor w2_packed, int64_t top_k, int64_t ffn_size,
                                           int64_t group_size, int64_t num_shared,
                                           std::optional<torch::Tensor> gate_bias) {
  check_cuda(x, "x");
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  auto xb = as_bf16_contig(x);
  auto gw = as_bf16_contig(gate_weight);
  const int64_t T = xb.size(0), d = xb.size(1), E = gw.size(0);
  torch::Tensor b;
  if (gate_bias.has_value() && gate_bias->defined()) b = gate_bias->to(torch::kFloat32).contiguous();
  auto y = torch::empty({T, d}, xb.options());
  auto ids = torch::empty({T, top_k}, xb.options().dtype(torch::kInt32));
  auto wts = torch::empty({T, top_k}, xb.options().dtype(torch::kFloat32));
  auto ws = workspace((int64_t)lmoe_moe_layer_workspace_bytes(T, (int)d, (int)ffn_size, (int)E, (int)top_k,
                                                               (int)num_shared),
                      xb);
  int st = lmoe_moe_layer_w4a16(xb.data_ptr(), T, (int)d, gw.data_ptr(), b.defined() ? b.data_ptr<float>() : nullptr,
                                (int)E, (int)top_k, (int)num_shared, w13_packed.data_ptr<uint8_t>(),
                                w2_packed.data_ptr<uint8_t>(), (int)ffn_size, (int)group_size, y.data_ptr(), ids.data_ptr<int32_t>(),
                                wts.data_ptr<float>(), ws.data_ptr(), ws.numel(), cur_stream());
  check_status(st, "moe_layer_w4a16");
  return {y, ids, wts};
}

// ---------------------------------------------------------------- gradients of grouped_gemm

// An uninitialised tensor beside `like`, straight from the allocator.
torch::Tensor empty_like_device(at::IntArrayRef sizes, torch::ScalarType type, const torch::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

void check_same_device(const torch::Tensor& t, const torch::Tensor& like, const char* name) {
  check_cuda(t, name);
  TORCH_CHECK(t.device() == like.device(), name, " must be on ", like.device(), ", is on ", t.device());
}

torch::Tensor check_offsets(const torch::Tensor& offsets, const torch::Tensor& like, int64_t num_experts) {
  check_same_device(offsets, like, "expert_offsets");
  TORCH_CHECK(num_experts >= 1, "num_experts must be at least 1");
  TORCH_CHECK(offsets.scalar_type() == torch::kInt64 || offsets.scalar_type() == torch::kInt32, "offsets int64/int32");
  TORCH_CHECK(offsets.numel() >= num_experts + 1, "expert_offsets must have num_experts + 1 entries");
  return offsets.contiguous();
}

void check_float(const torch::Tensor& t, const char* name) {
  const auto st = t.scalar_type();
  TORCH_CHECK(st == torch::kBFloat16 || st == torch::kFloat16 || st == torch::kFloat32, name,
              " must be bf16, fp16 or fp32, is ", st);
}

// The caller's error word, or none.
uint32_t* error_word(const std::optional<torch::Tensor>& error, const torch::Tensor& like) {
  if (!error.has_value() || !error->defined()) return nullptr;
  check_same_device(*error, like, "error");
  TORCH_CHECK(error->scalar_type() == torch::kInt32 && error->numel() == 1, "error must be one int32 value");
  return reinterpret_cast<uint32_t*>(error->data_ptr());
}

torch::Tensor grouped_gemm_dgrad(torch::Tensor grad_output, torch::Tensor weights, torch::Tensor expert_offsets,
                                 int64_t num_experts, std::optional<torch::Tensor> error) {
  check_cuda(grad_output, "grad_output");
  check_same_device(weights, grad_output, "weights");
  check_float(grad_output, "grad_output");
  TORCH_CHECK(grad_output.dim() == 2 && weights.dim() == 3, "grad_output [T,N], weights [E,N,K]");
  TORCH_CHECK(weights.size(0) >= num_experts && weights.size(1) == grad_output.size(1), "shape mismatch");
  TORCH_CHECK(weights.scalar_type() == grad_output.scalar_type(), "grad_output and weights differ in dtype");
  const at::AutoDispatchBelowADInplaceOrView below_autograd;   // no graph is recorded
  const c10::cuda::OptionalCUDAGuard guard(grad_output.device());
  auto off = check_offsets(expert_offsets, grad_output, num_experts);
  auto dy = contig16(grad_output);
  auto w = contig16(weights);
  const int64_t T = dy.size(0), N = w.size(1), K = w.size(2);
  check_sizes(T, N, K, num_experts);
  auto out = empty_like_device({T, K}, dy.scalar_type(), dy);
  const int dt = dtype_code(dy);
  auto ws = workspace((int64_t)lmoe_grouped_gemm_grad_workspace_bytes(0, dt, T, (int)N, (int)K, (int)num_experts), dy);
  check_status(lmoe_grouped_gemm_dgrad(dy.data_ptr(), dt, T, (int)N, w.data_ptr(), (int)K, off.data_ptr(),
                                       off.scalar_type() == torch::kInt64, (int)num_experts, out.data_ptr(),
                                       ws.data_ptr(), ws.numel(), error_word(error, dy), cur_stream()),
               "grouped_gemm_dgrad");
  return out;
}

torch::Tensor grouped_gemm_wgrad(torch::Tensor grad_output, torch::Tensor input, torch::Tensor expert_offsets,
                                 int64_t num_experts, std::optional<torch::ScalarType> out_dtype,
                                 std::optional<torch::Tensor> error) {
  check_cuda(grad_output, "grad_output");
  check_same_device(input, grad_output, "input");
  check_float(grad_output, "grad_output");
  TORCH_CHECK(grad_output.dim() == 2 && input.dim() == 2, "grad_output [T,N], input [T,K]");
  TORCH_CHECK(grad_output.size(0) == input.size(0), "grad_output and input differ in rows");
  TORCH_CHECK(input.scalar_type() == grad_output.scalar_type(), "grad_output and input differ in dtype");
  const auto ot = out_dtype.value_or(grad_output.scalar_type());
  TORCH_CHECK(ot == grad_output.scalar_type() || ot == torch::kFloat32, "out_dtype must be the operands' or float32");
  const at::AutoDispatchBelowADInplaceOrView below_autograd;   // no graph is recorded
  const c10::cuda::OptionalCUDAGuard guard(grad_output.device());
  auto off = check_offsets(expert_offsets, grad_output, num_experts);
  auto dy = contig16(grad_output);
  auto x = contig16(input);
  const int64_t T = dy.size(0), N = dy.size(1), K = x.size(1);
  check_sizes(T, N, K, num_experts);
  auto out = empty_like_device({num_experts, N, K}, ot, dy);
  const int dt = dtype_code(dy);
  auto ws = workspace((int64_t)lmoe_grouped_gemm_grad_workspace_bytes(1, dt, T, (int)N, (int)K, (int)num_experts), dy);
  check_status(lmoe_grouped_gemm_wgrad(dy.data_ptr(), dt, T, (int)N, x.data_ptr(), (int)K, off.data_ptr(),
                                       off.scalar_type() == torch::kInt64, (int)num_experts, dtype_code(out),
                                       out.data_ptr(), ws.data_ptr(), ws.numel(), error_word(error, dy), cur_stream()),
               "grouped_gemm_wgrad");
  return out;
}

// ---------------------------------------------------------------- microscaled 4-bit operands

int fp4_format(const std::string& format) {
  TORCH_CHECK(format == "mxfp4" || format == "nvfp4", "format must be 'mxfp4' or 'nvfp4', is '", format, "'");
  return format == "mxfp4" ? LMOE_FP4_MX : LMOE_FP4_NV;
}
int64_t fp4_block(int format) { return format == LMOE_FP4_MX ? 32 : 16; }

// The tensor scale(s) of `x` [.., rows, K]: one value, or one per leading index of a 3-D tensor.
// Returns the pointer and sets the rows that share a value.
const float* fp4_global_scale(const std::optional<torch::Tensor>& g, const torch::Tensor& x, int64_t lead,
                              int64_t rows, int format, int64_t* rows_per_scale) {
  *rows_per_scale = 1;
  if (!g.has_value() || !g->defined()) return nullptr;
  TORCH_CHECK(format == LMOE_FP4_NV, "global_scale belongs to nvfp4");
  check_same_device(*g, x, "global_scale");
  TORCH_CHECK(g->scalar_type() == torch::kFloat32 && g->is_contiguous(), "global_scale must be contiguous fp32");
  TORCH_CHECK(g->numel() == 1 || g->numel() == lead, "global_scale must have 1 or ", lead, " elements");
  if (rows > 0) *rows_per_scale = g->numel() == 1 ? rows : rows / lead;   // rows: lead is not 0 either
  return g->data_ptr<float>();
}

std::tuple<torch::Tensor, torch::Tensor> quantize_fp4(torch::Tensor x, const std::string& format,
                                                      std::optional<torch::Tensor> global_scale,
                                                      std::optional<torch::Tensor> positions) {
  check_cuda(x, "x");
  check_float(x, "x");
  const int fmt = fp4_format(format);
  TORCH_CHECK(x.dim() >= 2, "x must be [..., rows, K]");
  const int64_t K = x.size(-1);
  TORCH_CHECK(K > 0 && K % 32 == 0 && K <= INT32_MAX, "K must be a positive multiple of 32");
  const at::AutoDispatchBelowADInplaceOrView below_autograd;   // no graph is recorded
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  const bool strided = x.dim() == 2 && x.stride(1) == 1 && (x.size(0) <= 1 || x.stride(0) >= K);
  auto xc = strided ? x : x.contiguous();
  const int64_t rows = xc.numel() / K;
  const int64_t ldx = strided && x.size(0) > 1 ? x.stride(0) : K;
  int64_t rps = 1;
  const float* g = fp4_global_scale(global_scale, x, x.dim() == 3 ? x.size(0) : 1, rows, fmt, &rps);
  auto shape = x.sizes().vec();
  torch::Tensor pos;
  int64_t copies = 1, out_rows = rows;
  if (positions.has_value() && positions->defined()) {
    TORCH_CHECK(x.dim() == 2, "positions needs x [rows, K]");
    check_same_device(*positions, x, "positions");
    TORCH_CHECK(positions->scalar_type() == torch::kInt32, "positions must be int32");
    TORCH_CHECK(rows == 0 ? positions->numel() == 0 : (positions->numel() % rows == 0 && positions->numel() > 0),
                "positions must hold the same number of entries for each row");
    pos = positions->contiguous();
    copies = rows ? pos.numel() / rows : 1;
    out_rows = pos.numel();
    shape[0] = out_rows;
  }
  shape.back() = K / 2;
  auto q = empty_like_device(shape, torch::kUInt8, x);
  shape.back() = lmoe_fp4_scale_pitch((int)K, fmt);
  auto s = empty_like_device(shape, torch::kUInt8, x);
  if (rows > 0)
    check_status(lmoe_quantize_fp4(xc.data_ptr(), dtype_code(xc), rows, (int)K, ldx, fmt, g, rps,
                                   pos.defined() ? pos.data_ptr<int32_t>() : nullptr, (int)copies, out_rows,
                                   q.data_ptr<uint8_t>(), s.data_ptr<uint8_t>(), cur_stream()),
                 "quantize_fp4");
  // the columns of the scale rows, without the padding (in place: a view costs the host a microsecond)
  const auto strides = s.strides().vec();
  shape.back() = K / fp4_block(fmt);
  s.unsafeGetTensorImpl()->set_sizes_and_strides(shape, strides);
  return {q, s};
}

struct Fp4Operand {
  torch::Tensor q, s;
  int64_t pitch = 0;
};

// Codes contiguous and aligned; scale rows on a pitch of a multiple of 32 bytes with the whole
// padded row inside the storage, copied to such rows if they are not.
Fp4Operand fp4_operand(const torch::Tensor& q, const torch::Tensor& s, const torch::Tensor& like, int fmt, bool pad,
                       const char* name) {
  check_same_device(q, like, name);
  check_same_device(s, like, name);
  TORCH_CHECK(q.scalar_type() == torch::kUInt8 && s.scalar_type() == torch::kUInt8, name,
              ": codes and scales must be uint8");
  TORCH_CHECK(q.dim() >= 2 && q.dim() == s.dim(), name, ": codes [..., rows, K/2], scales [..., rows, K/block]");
  const int64_t K = q.size(-1) * 2;
  TORCH_CHECK(K > 0 && K % 32 == 0 && K <= INT32_MAX, name, ": K must be a positive multiple of 32");
  for (int64_t i = 0; i + 1 < q.dim(); ++i) TORCH_CHECK(q.size(i) == s.size(i), name, ": scales shape mismatch");
  TORCH_CHECK(s.size(-1) == K / fp4_block(fmt), name, ": scales shape mismatch");
  Fp4Operand o;
  o.q = contig16(q);
  const int64_t padded = lmoe_fp4_scale_pitch((int)K, fmt);
  const int64_t rows = q.numel() / (K / 2);
  if (rows == 0) {
    o.s = s;
    o.pitch = padded;
    return o;
  }
  // rows evenly spaced over all leading dimensions
  bool even = s.size(-1) == 1 || s.stride(-1) == 1;
  int64_t pitch = -1;   // of the innermost dimension with more than one row
  int64_t span = 0;
  for (int64_t i = s.dim() - 2; i >= 0 && even; --i) {
    if (s.size(i) == 1) continue;
    if (pitch < 0)
      pitch = s.stride(i);   // 0 where the rows are one broadcast row
    else
      even = s.stride(i) == span;
    span = s.stride(i) * s.size(i);
  }
  if (pitch < 0) pitch = padded;
  const int64_t have = (int64_t)s.storage().nbytes() - s.storage_offset();
  const bool fits = even && (reinterpret_cast<uintptr_t>(s.data_ptr()) % 32 == 0) &&
                    (pad ? pitch % 32 == 0 && pitch >= padded && (rows - 1) * pitch + padded <= have
                         : pitch >= s.size(-1));
  if (fits) {
    o.s = s;
    o.pitch = pitch;
  } else {
    auto shape = s.sizes().vec();
    shape.back() = padded;
    o.s = torch::zeros(shape, s.options());
    o.s.narrow(-1, 0, K / fp4_block(fmt)).copy_(s);
    o.pitch = padded;
  }
  return o;
}

torch::Tensor dequantize_fp4(torch::Tensor q, torch::Tensor scales, const std::string& format,
                             std::optional<torch::Tensor> global_scale) {
  check_cuda(q, "q");
  const int fmt = fp4_format(format);
  const at::AutoDispatchBelowADInplaceOrView below_autograd;   // no graph is recorded
  const c10::cuda::OptionalCUDAGuard guard(q.device());
  const Fp4Operand o = fp4_operand(q, scales, q, fmt, false, "q");
  const int64_t K = q.size(-1) * 2, rows = q.numel() / (K / 2);
  int64_t rps = 1;
  const float* g = fp4_global_scale(global_scale, q, q.dim() == 3 ? q.size(0) : 1, rows, fmt, &rps);
  auto shape = q.sizes().vec();
  shape.back() = K;
  auto out = empty_like_device(shape, torch::kBFloat16, q);
  if (rows > 0)
    check_status(lmoe_dequantize_fp4(o.q.data_ptr<uint8_t>(), o.s.data_ptr<uint8_t>(), o.pitch, rows, (int)K, fmt, g,
                                     rps, out.data_ptr(), cur_stream()),
                 "dequantize_fp4");
  return out;
}

const float* fp4_alpha(const std::optional<torch::Tensor>& alpha, const torch::Tensor& like, int64_t num_experts,
                       const char* name) {
  if (!alpha.has_value() || !alpha->defined()) return nullptr;
  check_same_device(*alpha, like, name);
  TORCH_CHECK(alpha->scalar_type() == torch::kFloat32 && alpha->is_contiguous() && alpha->numel() >= num_experts, name,
              " must be contiguous fp32 with num_experts elements");
  return alpha->data_ptr<float>();
}

torch::Tensor fp4_grouped_gemm(torch::Tensor input, torch::Tensor input_scales, torch::Tensor weights,
                               torch::Tensor weight_scales, torch::Tensor expert_offsets, int64_t num_experts,
                               const std::string& format, std::optional<torch::Tensor> alpha,
                               std::optional<torch::Tensor> weights_up, std::optional<torch::Tensor> weight_scales_up,
                               std::optional<torch::Tensor> alpha_up, std::optional<torch::ScalarType> out_dtype,
                               std::optional<torch::Tensor> error) {
  check_cuda(input, "input");
  const int fmt = fp4_format(format);
  TORCH_CHECK(input.dim() == 2 && weights.dim() == 3, "input [T,K/2], weights [E,N,K/2]");
  TORCH_CHECK(weights.size(0) >= num_experts && weights.size(2) == input.size(1), "shape mismatch");
  const at::AutoDispatchBelowADInplaceOrView below_autograd;   // no graph is recorded
  const c10::cuda::OptionalCUDAGuard guard(input.device());
  auto off = check_offsets(expert_offsets, input, num_experts);
  const Fp4Operand x = fp4_operand(input, input_scales, input, fmt, true, "input");
  const Fp4Operand w = fp4_operand(weights, weight_scales, input, fmt, true, "weights");
  Fp4Operand u;
  const bool swiglu = weights_up.has_value() && weights_up->defined();
  TORCH_CHECK(swiglu == (weight_scales_up.has_value() && weight_scales_up->defined()),
              "weights_up and weight_scales_up belong together");
  TORCH_CHECK(swiglu || !(alpha_up.has_value() && alpha_up->defined()), "alpha_up needs weights_up");
  Fp4Operand wp = w;
  if (swiglu) {
    TORCH_CHECK(weights_up->sizes() == weights.sizes(), "gate and up shapes differ");
    u = fp4_operand(*weights_up, *weight_scales_up, input, fmt, true, "weights_up");
    if (u.pitch != w.pitch) {   // one pitch for both: padded copies
      const int64_t nb = weight_scales.size(-1), padded = lmoe_fp4_scale_pitch((int)(input.size(1) * 2), fmt);
      for (Fp4Operand* o : {&wp, &u}) {
        if (o->pitch == padded) continue;
        auto shape = weight_scales.sizes().vec();
        shape.back() = padded;
        auto c = torch::zeros(shape, weight_scales.options());
        c.narrow(-1, 0, nb).copy_(o == &wp ? weight_scales : *weight_scales_up);
        o->s = c;
        o->pitch = padded;
      }
    }
  }
  const int64_t T = input.size(0), K = input.size(1) * 2, N = weights.size(1);
  check_sizes(T, N, K, num_experts);
  const float* al = fp4_alpha(alpha, input, num_experts, "alpha");
  const float* au = fp4_alpha(alpha_up, input, num_experts, "alpha_up");
  const auto ot = out_dtype.value_or(torch::kBFloat16);
  TORCH_CHECK(ot == torch::kBFloat16 || ot == torch::kFloat16 || ot == torch::kFloat32,
              "out_dtype must be bf16, fp16 or fp32");
  uint32_t* err = error_word(error, input);
  auto out = empty_like_device({T, N}, ot, input);
  if (T > 0 && N > 0)
    check_status(lmoe_fp4_grouped_gemm(x.q.data_ptr<uint8_t>(), x.s.data_ptr<uint8_t>(), x.pitch, T, (int)K,
                                       wp.q.data_ptr<uint8_t>(), wp.s.data_ptr<uint8_t>(),
                                       swiglu ? u.q.data_ptr<uint8_t>() : nullptr,
                                       swiglu ? u.s.data_ptr<uint8_t>() : nullptr, wp.pitch, (int)N, fmt,
                                       off.data_ptr(), off.scalar_type() == torch::kInt64, (int)num_experts, al, au,
                                       dtype_code(out), out.data_ptr(), err, cur_stream()),
                 "fp4_grouped_gemm");
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "light-moe operator surface on B200 (sm_100a): router, grouped GEMMs, W4A16 MoE layer";
  m.def("grouped_gemm", &grouped_gemm, "Grouped GEMM for MoE experts (bf16, offsets read on the device)",
        py::arg("input"), py::arg("weights"), py::arg("expert_offsets"), py::arg("num_experts"));
  m.def("fused_gate_topk", &fused_gate_topk, "Gate projection + softmax + top-k in one kernel",
        py::arg("hidden_states"), py::arg("gate_weight"), py::arg("top_k"));
  m.def("fused_gate_topk_permute", &fused_gate_topk_permute,
        "Gate + top-k + counts/offsets/stable permutation + row gather", py::arg("hidden_states"),
        py::arg("gate_weight"), py::arg("top_k"));
  m.def("fused_gate_topk_ex", &fused_gate_topk_ex,
        "Router with fp32 weights, int32 counts/offsets/sorted_idx and optional logits / probabilities",
        py::arg("hidden_states"), py::arg("gate_weight"), py::arg("top_k"), py::arg("bias") = py::none(),
        py::arg("return_logits") = false, py::arg("return_probs") = false);
  m.def("quantize_w4", &quantize_w4, "Symmetric per-group int4 quantisation", py::arg("w"), py::arg("group_size"));
  m.def("dequantize_w4", &dequantize_w4, "int4 -> bf16", py::arg("qweight"), py::arg("scales"),
        py::arg("group_size"));
  m.def("prepack_w4", &prepack_w4, "Canonical int4 -> GEMM device layout", py::arg("qweight"), py::arg("scales"),
        py::arg("group_size"), py::arg("qweight_up") = py::none(), py::arg("scales_up") = py::none());
  m.def("w4a16_grouped_gemm", &w4a16_grouped_gemm, "W4A16 grouped GEMM", py::arg("input"), py::arg("packed"),
        py::arg("expert_offsets"), py::arg("num_experts"), py::arg("N"),
        py::arg("group_size"), py::arg("epilogue") = 0, py::arg("dest_rows") = py::none(),
        py::arg("row_scale") = py::none(), py::arg("out_rows") = 0, py::arg("max_rows_per_expert") = 0,
        py::arg("segment_expert") = py::none());
  m.def("grouped_gemm_dgrad", &grouped_gemm_dgrad, "Input gradient of grouped_gemm", py::arg("grad_output"),
        py::arg("weights"), py::arg("expert_offsets"), py::arg("num_experts"), py::arg("error") = py::none());
  m.def("grouped_gemm_wgrad", &grouped_gemm_wgrad, "Weight gradient of grouped_gemm", py::arg("grad_output"),
        py::arg("input"), py::arg("expert_offsets"), py::arg("num_experts"), py::arg("out_dtype") = py::none(),
        py::arg("error") = py::none());
  m.def("quantize_fp4", &quantize_fp4, "Rows -> microscaled 4-bit floating point", py::arg("x"), py::arg("format"),
        py::arg("global_scale") = py::none(), py::arg("positions") = py::none());
  m.def("dequantize_fp4", &dequantize_fp4, "Microscaled 4-bit floating point -> bf16", py::arg("q"),
        py::arg("scales"), py::arg("format"), py::arg("global_scale") = py::none());
  m.def("fp4_grouped_gemm", &fp4_grouped_gemm, "Grouped GEMM of microscaled 4-bit operands", py::arg("input"),
        py::arg("input_scales"), py::arg("weights"), py::arg("weight_scales"), py::arg("expert_offsets"),
        py::arg("num_experts"), py::arg("format"), py::arg("alpha") = py::none(), py::arg("weights_up") = py::none(),
        py::arg("weight_scales_up") = py::none(), py::arg("alpha_up") = py::none(),
        py::arg("out_dtype") = py::none(), py::arg("error") = py::none());
  m.def("combine_rows", &combine_rows, "Weighted combine of slot rows back to tokens", py::arg("rows"),
        py::arg("positions"), py::arg("weights"), py::arg("num_tokens"), py::arg("top_k"),
        py::arg("extra_rows") = py::none(), py::arg("num_extra") = 0);
  m.def("moe_layer_w4a16", &moe_layer_w4a16, "W4A16 MoE layer", py::arg("x"), py::arg("gate_weight"),
        py::arg("w13_packed"), py::arg("w2_packed"), py::arg("top_k"),
        py::arg("ffn_size"), py::arg("group_size"), py::arg("num_shared") = 0, py::arg("gate_bias") = py::none());
}
