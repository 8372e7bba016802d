"""MoE layer with microscaled 4-bit experts and activations.

``FP4Experts`` holds the expert weights as ``ops.quantize_fp4`` writes them and ``FP4MoELayer`` is
the counterpart of ``layer.W4A16MoELayer`` (light-moe's ``SparseMoEBlock``,
python/light_moe/model/moe_block.py:63-169) whose expert products run on the block-scaled tensor
cores with both operands in 4 bits: route, quantise the tokens straight into expert order, gate /
up product with SwiGLU, quantise, down product, weighted combine.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import torch

from . import ops
from .layer import HostBufferCalls

# An nvfp4 tensor whose largest value is 448 * 6 needs no tensor scale.
NVFP4_RANGE = 448.0 * 6.0


@torch.no_grad()
def nvfp4_global_scale(x: torch.Tensor) -> torch.Tensor:
    """The tensor scale that maps the largest magnitude of ``x`` (of each x[i] of a 3-D tensor) to
    the end of nvfp4's range: fp32 [1] or [x.shape[0]]; 1 where everything is zero."""
    top = x.abs().amax(dim=(1, 2)) if x.dim() == 3 else x.abs().amax().reshape(1)
    g = top.float() / NVFP4_RANGE
    return torch.where(g > 0, g, torch.ones_like(g)).contiguous()


@dataclass
class FP4Experts:
    """Quantised experts: ``num_experts`` routed experts followed by ``num_shared``.  Codes
    [E, rows, K/2] and scales [E, rows, K/block] of gate (w1), up (w3) and down (w2), and their
    tensor scales fp32 [E] (None for mxfp4)."""

    format: str
    w1: Tuple[torch.Tensor, torch.Tensor]
    w3: Tuple[torch.Tensor, torch.Tensor]
    w2: Tuple[torch.Tensor, torch.Tensor]
    g1: Optional[torch.Tensor]
    g3: Optional[torch.Tensor]
    g2: Optional[torch.Tensor]
    num_experts: int
    num_shared: int
    hidden_size: int
    ffn_size: int

    @classmethod
    @torch.no_grad()
    def from_dense(cls, w1: torch.Tensor, w3: torch.Tensor, w2: torch.Tensor, format: str = "nvfp4",
                   shared: Optional[Sequence[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]]] = None) -> "FP4Experts":
        """Quantise dense expert weights on the GPU: w1, w3 [E, ffn, d] (gate, up), w2 [E, d, ffn];
        ``shared``: list of (w1, w3, w2) of always-on experts, as ``W4A16Experts.from_dense``."""
        E, F, d = w1.shape
        if w3.shape != w1.shape or w2.shape != (E, d, F):
            raise ValueError("w1 and w3 must be [E, ffn, d], w2 [E, d, ffn]")
        if d % 32 or F % 32:
            raise ValueError("hidden and ffn sizes must be multiples of 32")
        if shared:
            w1 = torch.cat([w1] + [s[0].unsqueeze(0) for s in shared])
            w3 = torch.cat([w3] + [s[1].unsqueeze(0) for s in shared])
            w2 = torch.cat([w2] + [s[2].unsqueeze(0) for s in shared])
        gs = [nvfp4_global_scale(w) if format == "nvfp4" else None for w in (w1, w3, w2)]
        qs = [ops.quantize_fp4(w, format, g) for w, g in zip((w1, w3, w2), gs)]
        return cls(format, *qs, *gs, E, w1.shape[0] - E, d, F)


class FP4MoELayer(HostBufferCalls, torch.nn.Module):
    """y = sum_j w_j * expert_{e_j}(x) (+ shared experts) with 4-bit experts and activations.

    ``input_scale`` / ``hidden_scale``: nvfp4 tensor scales (fp32, one value) of the tokens and of
    the experts' hidden rows, from a calibration; None = 1, which suits blocks whose largest value
    lies between about 0.1 and 2688.  They are buffers: values copied into them hold from the next
    call (or graph replay) on."""

    def __init__(self, gate_weight: torch.Tensor, experts: FP4Experts, top_k: int,
                 gate_bias: Optional[torch.Tensor] = None, input_scale: Optional[torch.Tensor] = None,
                 hidden_scale: Optional[torch.Tensor] = None):
        super().__init__()
        e = experts
        if gate_weight.shape != (e.num_experts, e.hidden_size):
            raise ValueError("gate_weight must be [num_experts, hidden_size]")
        if e.hidden_size % 64:
            raise ValueError("the router takes hidden sizes that are multiples of 64")
        if e.format != "nvfp4" and (input_scale is not None or hidden_scale is not None):
            raise ValueError("input_scale and hidden_scale belong to nvfp4")
        self.register_buffer("gate_weight", gate_weight.detach().to(torch.bfloat16).contiguous())
        self.register_buffer("gate_bias", None if gate_bias is None else gate_bias.detach().float().contiguous())
        one = lambda s: None if s is None else s.detach().to(gate_weight.device, torch.float32).reshape(1).contiguous()
        self.register_buffer("input_scale", one(input_scale))
        self.register_buffer("hidden_scale", one(hidden_scale))
        self.experts = e
        self.top_k = int(top_k)

    def _apply(self, fn, *args, **kwargs):
        # a move to another device takes the scales along, a cast leaves them in fp32
        scales = {n: b for n, b in self._buffers.items() if b is not None and n in ("input_scale", "hidden_scale")}
        super()._apply(fn, *args, **kwargs)
        for name, scale in scales.items():
            if self._buffers[name].dtype != torch.float32:
                self._buffers[name] = scale.to(self._buffers[name].device)
        return self

    def _load_from_state_dict(self, state_dict, prefix, *args, **kwargs):
        for name in ("_alpha1", "_alpha2", "_alpha3"):   # factors that earlier layers saved beside their scales
            state_dict.pop(prefix + name, None)
        super()._load_from_state_dict(state_dict, prefix, *args, **kwargs)

    def forward(self, x: torch.Tensor, return_routing: bool = False):
        e, k = self.experts, self.top_k
        shape = x.shape
        x2 = x.reshape(-1, shape[-1]).to(torch.bfloat16)
        T = x2.shape[0]
        if T == 0:
            y = x2.new_empty(shape)
            return (y, x2.new_empty((0, k), dtype=torch.int32), x2.new_empty((0, k), dtype=torch.float32)) \
                if return_routing else y
        ids, weights, _, offsets, _, positions = ops.fused_gate_topk_ex(x2, self.gate_weight, k, self.gate_bias)[:6]
        positions, combine, segments, slots = positions.view(T, k), weights, e.num_experts, k
        if e.num_shared:
            # shared expert s: rows T * k + s * T + t of every token t, weight 1
            S, dev = e.num_shared, x2.device
            base = T * k + T * torch.arange(S + 1, dtype=torch.int32, device=dev)
            positions = torch.cat([positions, base[:S] + torch.arange(T, dtype=torch.int32, device=dev)[:, None]], 1)
            offsets = torch.cat([offsets[:-1], base])
            combine = torch.cat([weights, weights.new_ones(T, S)], 1)
            segments, slots = segments + S, k + S
        # the products' factors, from the scales as they are now (a new calibration may have been copied in)
        times = lambda g, s: g if g is None or s is None else g * s
        xq, xs = ops.quantize_fp4(x2, e.format, self.input_scale, positions=positions.contiguous())
        h = ops.fp4_grouped_gemm(xq, xs, *e.w1, offsets, segments, e.format, alpha=times(e.g1, self.input_scale),
                                 weights_up=e.w3[0], weight_scales_up=e.w3[1],
                                 alpha_up=times(e.g3, self.input_scale))
        hq, hs = ops.quantize_fp4(h, e.format, self.hidden_scale)
        o = ops.fp4_grouped_gemm(hq, hs, *e.w2, offsets, segments, e.format, alpha=times(e.g2, self.hidden_scale))
        y = ops.combine_rows(o, positions, combine, T, slots).view(shape)
        return (y, ids, weights) if return_routing else y
