"""Training with the grouped products: an autograd function and the modules around it.

light-moe trains its experts through autograd of one ``mm`` per expert
(python/light_moe/ops/grouped_gemm.py:65-106, ``GroupedLinear`` :109-199, used three times by
``SparseMoEBlockFast``, python/light_moe/model/moe_block.py:179-274).  Here a grouped product is
one launch in each direction, with the row ranges read on the device:

* ``grouped_linear(input, weights, expert_offsets)``  rows [T, in] x weights [E, out, in] ->
  [T, out]; its backward is ``ops.grouped_gemm_dgrad`` and ``ops.grouped_gemm_wgrad``;
* ``GroupedLinear``   the module, weights ``[num_experts, out_features, in_features]``;
* ``GroupedExperts``  the SwiGLU experts of a MoE block on routed tokens, differentiable in the
  tokens, the routing weights and the expert weights.

bf16, fp16 and fp32, any sizes.  Nothing synchronises with the host, so forward and backward can
be captured in a CUDA graph; as for any captured backward pass, free (or detach) earlier eager
graphs of the same leaves first.
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import ops


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, weights, expert_offsets):
        ctx.save_for_backward(input, weights, expert_offsets)
        return ops.grouped_gemm(input, weights, expert_offsets, weights.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        input, weights, offsets = ctx.saved_tensors
        E = weights.shape[0]
        grad_input = grad_weights = None
        if ctx.needs_input_grad[0]:
            grad_input = ops.grouped_gemm_dgrad(grad_output, weights, offsets, E)
        if ctx.needs_input_grad[1]:
            grad_weights = ops.grouped_gemm_wgrad(grad_output, input, offsets, E)
        return grad_input, grad_weights, None


def grouped_linear(input: torch.Tensor, weights: torch.Tensor, expert_offsets: torch.Tensor) -> torch.Tensor:
    """Rows [expert_offsets[e], expert_offsets[e + 1]) of ``input`` [T, in] times ``weights[e]``
    [out, in] transposed -> [T, out]; rows outside every expert are zero (and get a zero gradient).
    Differentiable in ``input`` and ``weights``, once."""
    if input.dim() != 2 or weights.dim() != 3 or weights.shape[2] != input.shape[1]:
        raise ValueError("input must be [T, in_features] and weights [E, out_features, in_features]")
    if input.dtype != weights.dtype or input.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError("input and weights must share one of bf16, fp16, fp32")
    if expert_offsets.numel() != weights.shape[0] + 1:
        raise ValueError("expert_offsets must have num_experts + 1 entries")
    return _GroupedLinear.apply(input, weights, expert_offsets)


class GroupedLinear(torch.nn.Module):
    """``num_experts`` bias-free linear maps as one parameter [num_experts, out, in]
    (python/light_moe/ops/grouped_gemm.py:109-199)."""

    def __init__(self, num_experts: int, in_features: int, out_features: int, device=None, dtype=None):
        super().__init__()
        self.num_experts, self.in_features, self.out_features = num_experts, in_features, out_features
        self.weight = torch.nn.Parameter(torch.empty(num_experts, out_features, in_features, device=device,
                                                     dtype=dtype))
        self.reset_parameters()

    def reset_parameters(self) -> None:
        bound = 1.0 / math.sqrt(self.in_features)
        torch.nn.init.uniform_(self.weight, -bound, bound)

    def forward(self, input: torch.Tensor, expert_offsets: torch.Tensor) -> torch.Tensor:
        return grouped_linear(input, self.weight, expert_offsets)

    def extra_repr(self) -> str:
        return f"num_experts={self.num_experts}, in_features={self.in_features}, out_features={self.out_features}"


class GroupedExperts(torch.nn.Module):
    """y[t] = sum_j routing_weights[t, j] * down(silu(gate(x_t)) * up(x_t)) of expert
    expert_indices[t, j]: the experts of light-moe's ``SparseMoEBlockFast``
    (python/light_moe/model/moe_block.py:216-274), trainable."""

    def __init__(self, num_experts: int, hidden_size: int, intermediate_size: int, device=None, dtype=None):
        super().__init__()
        kw = dict(device=device, dtype=dtype)
        self.num_experts = num_experts
        self.gate_proj = GroupedLinear(num_experts, hidden_size, intermediate_size, **kw)
        self.up_proj = GroupedLinear(num_experts, hidden_size, intermediate_size, **kw)
        self.down_proj = GroupedLinear(num_experts, intermediate_size, hidden_size, **kw)

    def forward(self, hidden_states: torch.Tensor, expert_indices: torch.Tensor,
                routing_weights: torch.Tensor) -> torch.Tensor:
        """hidden_states [T, d]; expert_indices, routing_weights [T, k] (as the router gives them)."""
        if expert_indices.dim() != 2 or expert_indices.shape[1] < 1 or routing_weights.shape != expert_indices.shape \
                or hidden_states.dim() != 2 or hidden_states.shape[0] != expert_indices.shape[0]:
            raise ValueError("hidden_states must be [T, d], expert_indices and routing_weights [T, k]")
        T, k = expert_indices.shape
        flat = expert_indices.reshape(-1).long()
        ids, order = torch.sort(flat, stable=True)             # (expert, token, slot) order
        offsets = torch.searchsorted(ids, torch.arange(self.num_experts + 1, device=ids.device))
        rows = hidden_states[order // k]
        h = torch.nn.functional.silu(self.gate_proj(rows, offsets)) * self.up_proj(rows, offsets)
        out = self.down_proj(h, offsets).float() * routing_weights.reshape(-1)[order].float()[:, None]
        back = torch.empty_like(order)                         # the row of each (token, slot)
        back[order] = torch.arange(T * k, device=order.device)
        return out[back].view(T, k, out.shape[1]).sum(1).to(hidden_states.dtype)
