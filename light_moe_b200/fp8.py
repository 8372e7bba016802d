"""MoE layer with block-scaled 8-bit experts.

``FP8Experts`` holds the expert weights as ``ops.quantize_fp8(w, block_rows=128)`` writes them: E4M3 codes with
one fp32 scale per block of 128 x 128, the form that fine-grained MoE checkpoints are published in.
``FP8MoELayer`` is the counterpart of ``layer.W4A16MoELayer`` (light-moe's ``SparseMoEBlock``,
python/light_moe/model/moe_block.py:63-169) on them.  A few tokens (a decode step) run as
``ops.moe_layer_few_tokens``: two kernels that stream the chosen experts' weights, activations not quantised.
Larger batches run on the 8-bit tensor cores: route, quantise the tokens straight into expert order (one
scale per 128 values), gate / up product with SwiGLU, quantise, down product, weighted combine.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import torch

from . import ops
from .layer import HostBufferCalls

# Batches of at most FEW_TOKENS tokens, of a hidden size up to FEW_TOKENS_HIDDEN (where 8 tokens fit shared
# memory), take the few-token kernels.  Replayed, us, those against the kernels for larger batches: 8 experts of
# 4096 / 14336, two a token: 1 token 81 against 107, 4 177 against 193, 8 245 against 238, 12 352 against 256; 64 of 2048 /
# 1408, six a token and two shared: 1 38 against 76, 8 93 against 123, 12 144 against 131; 8 of 1024 / 2816: 8 39 against
# 47, 12 53 against 49.
FEW_TOKENS, FEW_TOKENS_HIDDEN = 8, 8192
FEW_TOKENS_FFN, FEW_TOKENS_SHARED = 65536, 16   # what those kernels take
# Experts that the router and one grouped product take.
MOST_EXPERTS = 256


@dataclass
class FP8Experts:
    """Quantised experts: ``num_experts`` routed experts followed by ``num_shared``.  Codes float8_e4m3fn
    [E, rows, K] and scales fp32 [E, ceil(rows / 128), ceil(K / 128)] of gate (w1), up (w3) and down (w2)."""

    w1: Tuple[torch.Tensor, torch.Tensor]
    w3: Tuple[torch.Tensor, torch.Tensor]
    w2: Tuple[torch.Tensor, torch.Tensor]
    num_experts: int
    num_shared: int
    hidden_size: int
    ffn_size: int

    @classmethod
    @torch.no_grad()
    def from_dense(cls, w1: torch.Tensor, w3: torch.Tensor, w2: torch.Tensor, power_of_two: bool = False,
                   shared: Optional[Sequence[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]]] = None) -> "FP8Experts":
        """Quantise dense expert weights on the GPU: w1, w3 [E, ffn, d] (gate, up), w2 [E, d, ffn];
        ``shared``: list of (w1, w3, w2) of always-on experts, as ``W4A16Experts.from_dense``."""
        E, F, d = w1.shape
        if w3.shape != w1.shape or w2.shape != (E, d, F):
            raise ValueError("w1 and w3 must be [E, ffn, d], w2 [E, d, ffn]")
        if shared:
            w1 = torch.cat([w1] + [s[0].unsqueeze(0) for s in shared])
            w3 = torch.cat([w3] + [s[1].unsqueeze(0) for s in shared])
            w2 = torch.cat([w2] + [s[2].unsqueeze(0) for s in shared])
        qs = [ops.quantize_fp8(w, block_rows=128, power_of_two=power_of_two) for w in (w1, w3, w2)]
        return cls.from_quantized(*qs, num_experts=E)

    @classmethod
    def from_quantized(cls, w1: Tuple[torch.Tensor, torch.Tensor], w3: Tuple[torch.Tensor, torch.Tensor],
                       w2: Tuple[torch.Tensor, torch.Tensor], num_experts: int) -> "FP8Experts":
        """From (codes, scales) of a checkpoint, routed experts first, then shared ones; value = code * scale."""
        Et, F, d = w1[0].shape
        if w3[0].shape != w1[0].shape or w2[0].shape != (Et, d, F) or not 1 <= num_experts <= Et:
            raise ValueError("w1 and w3 must be [E, ffn, d], w2 [E, d, ffn]")
        if d % 16 or F % 16:
            raise ValueError("hidden and ffn sizes must be multiples of 16")
        for q, s in (w1, w3, w2):
            if q.dtype != torch.float8_e4m3fn or s.dtype != torch.float32 \
                    or s.shape != (Et, -(-q.shape[1] // 128), -(-q.shape[2] // 128)):
                raise ValueError("codes must be float8_e4m3fn and scales fp32, one per block of 128 x 128")
        # laid out once as the kernels read them
        whole = lambda w: tuple(t.contiguous() for t in w)
        return cls(whole(w1), whole(w3), whole(w2), num_experts, Et - num_experts, d, F)


class FP8MoELayer(HostBufferCalls, torch.nn.Module):
    """y = sum_j w_j * expert_{e_j}(x) (+ shared experts) with 8-bit experts; activations in bf16 up to
    ``FEW_TOKENS`` tokens, in 8 bits beyond."""

    def __init__(self, gate_weight: torch.Tensor, experts: FP8Experts, top_k: int,
                 gate_bias: Optional[torch.Tensor] = None):
        super().__init__()
        e = experts
        if gate_weight.shape != (e.num_experts, e.hidden_size):
            raise ValueError("gate_weight must be [num_experts, hidden_size]")
        if e.hidden_size % 64:
            raise ValueError("the router takes hidden sizes that are multiples of 64")
        if gate_bias is not None and gate_bias.shape != (e.num_experts,):
            raise ValueError("gate_bias must be [num_experts]")
        if max(e.num_experts, e.num_shared) > MOST_EXPERTS:
            raise ValueError(f"at most {MOST_EXPERTS} routed experts, and as many shared ones")
        if not 1 <= top_k <= min(16, e.num_experts):
            raise ValueError("top_k must be 1 .. min(16, num_experts)")
        self.register_buffer("gate_weight", gate_weight.detach().to(torch.bfloat16).contiguous())
        self.register_buffer("gate_bias", None if gate_bias is None else gate_bias.detach().float().contiguous())
        self.experts = e
        self.top_k = int(top_k)

    def forward(self, x: torch.Tensor, return_routing: bool = False):
        e, k = self.experts, self.top_k
        shape = x.shape
        x2 = x.reshape(-1, shape[-1]).to(torch.bfloat16)
        T = x2.shape[0]
        if T == 0:
            y = x2.new_empty(shape)
            return (y, x2.new_empty((0, k), dtype=torch.int32), x2.new_empty((0, k), dtype=torch.float32)) \
                if return_routing else y
        if T <= FEW_TOKENS and e.hidden_size <= FEW_TOKENS_HIDDEN and e.ffn_size % 32 == 0 \
                and e.ffn_size <= FEW_TOKENS_FFN and e.num_shared <= FEW_TOKENS_SHARED:
            # (a cast of the module may have changed the router's types)
            y, ids, weights = ops.moe_layer_few_tokens(
                x2, self.gate_weight.to(torch.bfloat16), e.w1[0], e.w3[0], e.w2[0], k, w1_scales=e.w1[1],
                w3_scales=e.w3[1], w2_scales=e.w2[1], num_shared=e.num_shared,
                gate_bias=None if self.gate_bias is None else self.gate_bias.float())
            y = y.view(shape)
            return (y, ids, weights) if return_routing else y
        ids, weights, _, offsets, _, positions = ops.fused_gate_topk_ex(x2, self.gate_weight, k, self.gate_bias)[:6]
        positions, combine, segments, slots = positions.view(T, k), weights, e.num_experts, k
        apart = 0   # shared experts beyond what one product takes: they have products of their own
        if e.num_shared:
            # shared expert s: rows T * k + s * T + t of every token t, weight 1
            S, dev = e.num_shared, x2.device
            base = T * k + T * torch.arange(S + 1, dtype=torch.int32, device=dev)
            positions = torch.cat([positions, base[:S] + torch.arange(T, dtype=torch.int32, device=dev)[:, None]], 1)
            if segments + S > MOST_EXPERTS:
                apart = S
            else:
                offsets = torch.cat([offsets[:-1], base])
                combine = torch.cat([weights, weights.new_ones(T, S)], 1)
                segments, slots = segments + S, k + S
        xq, xs = ops.quantize_fp8(x2, positions=positions.contiguous())
        if apart:
            n, cut = T * k, lambda a, b: ((q[a:b], s[a:b]) for q, s in (e.w1, e.w3, e.w2))
            o = _products(xq[:n], xs[:n], offsets, segments, *cut(0, segments))
            extra = _products(xq[n:], xs[n:], base - n, apart, *cut(segments, segments + apart))
            y = ops.combine_rows(o, positions[:, :k], combine, T, k, extra, apart)
        else:
            o = _products(xq, xs, offsets, segments, e.w1, e.w3, e.w2)
            y = ops.combine_rows(o, positions, combine, T, slots)
        y = y.view(shape)
        return (y, ids, weights) if return_routing else y


def _products(xq: torch.Tensor, xs: torch.Tensor, offsets: torch.Tensor, experts: int, w1, w3, w2) -> torch.Tensor:
    """The rows between the offsets through their experts."""
    h = ops.fp8_grouped_gemm(xq, xs, *w1, offsets, experts, weights_up=w3[0], weight_scales_up=w3[1])
    hq, hs = ops.quantize_fp8(h)
    return ops.fp8_grouped_gemm(hq, hs, *w2, offsets, experts)
