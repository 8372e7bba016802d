"""The light-moe operator surface, backed by the sm_100a library.

Same names, argument names and return types as the reference's ``light_moe._C``
(csrc/bindings.cpp:28-49 of Whitehall945/light-moe):

    grouped_gemm(input, weights, expert_offsets, num_experts) -> Tensor
    fused_gate_topk(hidden_states, gate_weight, top_k) -> (ids int32, weights)
    fused_gate_topk_permute(hidden_states, gate_weight, top_k)
        -> (permuted, ids, weights, offsets int64, sorted_idx int64)

plus the new ops (``fused_gate_topk_ex``, ``quantize_w4``, ``dequantize_w4``, ``prepack_w4``,
``w4a16_grouped_gemm``, ``moe_layer_w4a16``; the gradients ``grouped_gemm_dgrad`` and
``grouped_gemm_wgrad``; the 4-bit floating point ``quantize_fp4``, ``dequantize_fp4`` and
``fp4_grouped_gemm``; the 8-bit ``quantize_fp8``, ``dequantize_fp8`` and ``fp8_grouped_gemm``;
``moe_layer_few_tokens``).  Every op runs the CUDA library; if the
``_C`` extension has not been built, calling any op raises -- there is no fallback path.
"""
from __future__ import annotations

import importlib

_ext = None


def extension():
    """The compiled ``_C`` module (raises RuntimeError if it is not built)."""
    global _ext
    if _ext is None:
        try:
            _ext = importlib.import_module("light_moe_b200._C")
        except ImportError as e:  # pragma: no cover - exercised only without a build
            raise RuntimeError(
                "light_moe_b200._C is not built; run `python -m light_moe_b200.build` "
                f"(import error: {e})") from e
    return _ext


def grouped_gemm(input, weights, expert_offsets, num_experts):
    """Dense grouped GEMM in the input dtype, any row length; rows outside every expert range are
    zero (grouped_gemm.cu:24).  fp32 rows whose length is not a multiple of 4 may give NaN where the
    sum is an infinity."""
    return extension().grouped_gemm(input, weights, expert_offsets, num_experts)


def fused_gate_topk(hidden_states, gate_weight, top_k):
    """(expert_ids int32 [T, k], expert_weights [T, k] in the hidden dtype)."""
    return extension().fused_gate_topk(hidden_states, gate_weight, top_k)


def fused_gate_topk_permute(hidden_states, gate_weight, top_k):
    """(permuted [T*k, d], ids, weights, expert_offsets int64 [E+1], sorted_idx int64 [T*k])."""
    return extension().fused_gate_topk_permute(hidden_states, gate_weight, top_k)


def fused_gate_topk_ex(hidden_states, gate_weight, top_k, bias=None, return_logits=False, return_probs=False):
    """[ids int32, weights fp32, counts int32, offsets int32, sorted_idx int32, positions int32
    (, logits fp32 [T, E]) (, probs fp32 [T, E])] -- positions is the inverse permutation of
    sorted_idx, probs the full softmax probabilities."""
    return extension().fused_gate_topk_ex(hidden_states, gate_weight, top_k, bias, return_logits, return_probs)


def quantize_w4(w, group_size):
    """w [..., N, K] -> (qweight uint8 [..., N, K/2], scales fp16 [..., N, K/group_size])."""
    return extension().quantize_w4(w, group_size)


def dequantize_w4(qweight, scales, group_size):
    """int4 -> bf16 [..., N, K]; bit-exact bf16_rn(q * s)."""
    return extension().dequantize_w4(qweight, scales, group_size)


def prepack_w4(qweight, scales, group_size, qweight_up=None, scales_up=None):
    """Canonical int4 [E, N, K/2] + scales -> the GEMM's streaming layout (scales embedded;
    paired with the up projection if given).  Returns one uint8 tensor."""
    return extension().prepack_w4(qweight, scales, group_size, qweight_up, scales_up)


def w4a16_grouped_gemm(input, packed, expert_offsets, num_experts, N, group_size,
                       epilogue=0, dest_rows=None, row_scale=None, out_rows=0, max_rows_per_expert=0,
                       segment_expert=None):
    """Grouped W4A16 GEMM over `num_experts` row segments (segment_expert maps segment -> weights)."""
    return extension().w4a16_grouped_gemm(input, packed, expert_offsets, num_experts, N,
                                          group_size, epilogue, dest_rows, row_scale, out_rows,
                                          max_rows_per_expert, segment_expert)


def grouped_gemm_dgrad(grad_output, weights, expert_offsets, num_experts, error=None):
    """Input gradient of grouped_gemm: [T, N] x [E, N, K] -> [T, K] (rows outside every expert are
    zero).  bf16 / fp16 on tensor cores, fp32 in fp32 accuracy (values below 2**-107 to 2**-134; NaN
    where the sum may be an infinity); any N, K; operands of one dtype.

    Offsets that decrease or leave [0, T] put every row outside the experts.  ``error``: one int32
    value on the device, zeroed by the caller (None: nobody asks); such offsets and a kernel that gave
    up waiting, whose output is not whole, set it.  Nothing waits for the device to look at it."""
    return extension().grouped_gemm_dgrad(grad_output, weights, expert_offsets, num_experts, error)


def grouped_gemm_wgrad(grad_output, input, expert_offsets, num_experts, out_dtype=None, error=None):
    """Weight gradient of grouped_gemm: sum over each expert's rows of grad_output^T input ->
    [E, N, K] in the operands' dtype or, with ``out_dtype=torch.float32``, as the fp32 sums; experts
    without rows are zero.  Sums of 16-bit products truncate where they add: of one sign they come out
    low by 2.5e-5 of their value after 8192 rows, 3.4e-4 after 65536 (fp32 operands: no such loss).
    ``error`` as for the input gradient."""
    return extension().grouped_gemm_wgrad(grad_output, input, expert_offsets, num_experts, out_dtype, error)


def quantize_fp4(x, format, global_scale=None, positions=None):
    """x [..., K] (bf16 / fp16 / fp32, K % 32 == 0) -> (codes uint8 [..., K/2], scales uint8
    [..., K/block]): E2M1 values, two to a byte (even column low), under one scale byte per
    block -- ``"mxfp4"`` E8M0 scales for blocks of 32, ``"nvfp4"`` E4M3 scales for blocks of 16
    times ``global_scale`` (fp32, one value or one per leading index of a 3-D x; None = 1).
    Round to nearest even, saturating; blocks with an infinity or NaN read back as NaN.

    ``positions`` int32 [rows, copies] (a permutation of 0 .. rows * copies - 1, like the
    router's inverse permutation): row r is written to rows positions[r, :], so a MoE layer's
    permutation needs no pass of its own.  Scale rows lie on a pitch of a multiple of 32 bytes
    (the returned tensor is a view); the product copies scales that do not."""
    return extension().quantize_fp4(x, format, global_scale, positions)


def dequantize_fp4(q, scales, format, global_scale=None):
    """Codes and scales -> bf16 [..., K]: bf16_rn(fp32_rn(code * scale * global_scale))."""
    return extension().dequantize_fp4(q, scales, format, global_scale)


def fp4_grouped_gemm(input, input_scales, weights, weight_scales, expert_offsets, num_experts, format,
                     alpha=None, weights_up=None, weight_scales_up=None, alpha_up=None, out_dtype=None, error=None):
    """Grouped product of 4-bit operands (codes and scales as quantize_fp4 returns them): rows
    [T, K] x weights [E, N, K] -> [T, N] of ``out_dtype`` (bf16 by default), times ``alpha[e]``
    (fp32 [E], the product of the operands' global scales).  With ``weights_up``:
    silu(gate) * up.  Exact products, fp32 sums (truncated where they add, 2e-6 low after 14336 products
    of one sign under nvfp4); rows outside every expert are zero.
    ``error`` as for grouped_gemm_dgrad."""
    return extension().fp4_grouped_gemm(input, input_scales, weights, weight_scales, expert_offsets, num_experts,
                                        format, alpha, weights_up, weight_scales_up, alpha_up, out_dtype, error)


def quantize_fp8(x, block_rows=1, power_of_two=False, positions=None):
    """x [..., rows, K] (bf16 / fp16 / fp32, K % 16 == 0) -> (codes float8_e4m3fn [..., rows, K], scales fp32
    [..., rows / block_rows, K / 128], both rounded up): one scale per 128 columns of a row (``block_rows=1``,
    activations) or per block of 128 x 128 (``block_rows=128``, weights).

    scale = max(max|x| / 448, 2**-126), rounded up to a power of two with ``power_of_two``; codes are the
    nearest E4M3 values of x / scale, ties to even; blocks with an infinity or NaN read back as NaN.
    Scales of rows lie block after block (the returned tensor is a view with stride 1 along the rows).

    ``positions`` (``block_rows=1``) int32 [rows, copies] (a permutation of 0 .. rows * copies - 1): row r
    is written to rows positions[r, :], as for ``quantize_fp4``."""
    return extension().quantize_fp8(x, block_rows, power_of_two, positions)


def dequantize_fp8(q, scales, block_rows=1, out_dtype=None):
    """Codes and scales (any strides) -> ``out_dtype`` (bf16 by default) [..., rows, K]:
    rn(fp32_rn(code * scale))."""
    return extension().dequantize_fp8(q, scales, block_rows, out_dtype)


def fp8_grouped_gemm(input, input_scales, weights, weight_scales, expert_offsets, num_experts, weights_up=None,
                     weight_scales_up=None, out_dtype=None, error=None):
    """Grouped product of 8-bit operands (codes and scales as quantize_fp8 returns them): rows [T, K] with
    scales [T, K / 128] x weights [E, N, K] with scales [E, N / 128, K / 128] -> [T, N] of ``out_dtype`` (bf16 by
    default).  With ``weights_up``: silu(gate) * up.  Exact products, fp32 sums; rows outside every expert
    are zero.  Scales of rows that do not have stride 1 along the rows are copied.  ``error`` as for
    grouped_gemm_dgrad."""
    return extension().fp8_grouped_gemm(input, input_scales, weights, weight_scales, expert_offsets, num_experts,
                                        weights_up, weight_scales_up, out_dtype, error)


def combine_rows(rows, positions, weights, num_tokens, top_k, extra_rows=None, num_extra=0):
    """y[t] = sum_j weights[t,j] * rows[positions[t,j]] + sum_s extra_rows[s*T + t]."""
    return extension().combine_rows(rows, positions, weights, num_tokens, top_k, extra_rows, num_extra)


def moe_layer_w4a16(x, gate_weight, w13_packed, w2_packed, top_k, ffn_size, group_size, num_shared=0,
                    gate_bias=None):
    """[y bf16 [T, d], ids int32 [T, k], weights fp32 [T, k]]."""
    return extension().moe_layer_w4a16(x, gate_weight, w13_packed, w2_packed, top_k, ffn_size, group_size,
                                       num_shared, gate_bias)


def moe_layer_few_tokens(x, gate_weight, w1, w3, w2, top_k, w1_scales=None, w3_scales=None, w2_scales=None,
                         num_shared=0, gate_bias=None):
    """[y [T, d] in x's dtype, ids int32 [T, k], weights fp32 [T, k]]: the whole MoE layer (router, SwiGLU
    experts, weighted sum) for at most 16 tokens, in two kernels.

    x [T, d] and gate_weight [E, d] bf16 or fp16 (the same); w1, w3 [E + S, ffn, d] and w2 [E + S, d, ffn] of
    that dtype, or float8_e4m3fn with the scales of ``quantize_fp8(w, block_rows=128)``; the last
    ``num_shared`` experts take every token with weight 1; gate_bias fp32 [E].  The activations are not
    quantised.  d % 64 == 0, ffn % 32 == 0."""
    return extension().moe_layer_few_tokens(x, gate_weight, w1, w3, w2, top_k, w1_scales, w3_scales, w2_scales,
                                            num_shared, gate_bias)
