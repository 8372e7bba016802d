"""GPU tests of the MoE layer with 4-bit experts: its steps together, against the steps called one
by one, and each product against 64 bits on the operands that it got."""
import numpy as np
import pytest
import torch

import fp4_reference as ref
from light_moe_b200 import ops
from light_moe_b200.fp4 import FP4Experts, FP4MoELayer, nvfp4_global_scale

pytestmark = pytest.mark.gpu


def _make(T, d, F, E, k, fmt, S=0, seed=0, scales=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x = r(T, d).to(torch.bfloat16)
    w1, w3, w2 = r(E + S, F, d) * 0.05, r(E + S, F, d) * 0.05, r(E + S, d, F) * 0.05
    shared = [(w1[E + s], w3[E + s], w2[E + s]) for s in range(S)] or None
    ex = FP4Experts.from_dense(w1[:E], w3[:E], w2[:E], fmt, shared=shared)
    kw = dict(input_scale=torch.tensor(0.002), hidden_scale=torch.tensor([0.0005])) if scales else {}
    gate = r(E, d) * 0.05
    return x, FP4MoELayer(gate, ex, k, **kw), (w1, w3, w2)


def _by_hand(mod, x, T, k):
    """The layer without the permutation inside the quantiser: gather, then quantise."""
    e = mod.experts
    ids, w, _, off, sidx, pos = ops.fused_gate_topk_ex(x, mod.gate_weight, k, mod.gate_bias)[:6]
    rows = x[(sidx // k).long()]
    bounds = off
    if e.num_shared:
        rows = torch.cat([rows] + [x] * e.num_shared)
        bounds = torch.cat([off, off[-1:] + T * torch.arange(1, e.num_shared + 1, device="cuda", dtype=torch.int32)])
    n = e.num_experts + e.num_shared
    xq, xs = ops.quantize_fp4(rows, e.format, mod.input_scale)
    gx = 1.0 if mod.input_scale is None else mod.input_scale
    gh = 1.0 if mod.hidden_scale is None else mod.hidden_scale
    al = lambda g, s: None if g is None else g * s
    h = ops.fp4_grouped_gemm(xq, xs, *e.w1, bounds, n, e.format, alpha=al(e.g1, gx), weights_up=e.w3[0],
                             weight_scales_up=e.w3[1], alpha_up=al(e.g3, gx))
    hq, hs = ops.quantize_fp4(h, e.format, mod.hidden_scale)
    o = ops.fp4_grouped_gemm(hq, hs, *e.w2, bounds, n, e.format, alpha=al(e.g2, gh))
    y = torch.zeros(T, x.shape[1], device="cuda")
    for j in range(k):
        y = y + w[:, j:j + 1] * o[pos.view(T, k)[:, j].long()].float()
    for s in range(e.num_shared):
        y = y + o[T * k + s * T:T * k + (s + 1) * T].float()
    return y.to(torch.bfloat16), ids, w


@pytest.mark.parametrize("fmt,scales", [("mxfp4", False), ("nvfp4", False), ("nvfp4", True)])
@pytest.mark.parametrize("T,d,F,E,k,S", [(1, 256, 128, 8, 2, 0), (37, 256, 96, 8, 2, 0), (300, 128, 160, 16, 4, 2),
                                         (1500, 256, 256, 4, 2, 1)])
def test_layer_equals_its_steps(fmt, scales, T, d, F, E, k, S):
    x, mod, _ = _make(T, d, F, E, k, fmt, S, seed=T, scales=scales)
    y, ids, w = mod(x, return_routing=True)
    want, ids2, w2 = _by_hand(mod, x, T, k)
    assert torch.equal(ids, ids2) and torch.equal(w, w2)
    assert torch.equal(y, want)
    assert torch.equal(mod(x.view(1, T, d)).view(T, d), y)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_layer_is_near_the_dense_experts(fmt):
    """Errors of independent roundings: an E2M1 value is off by at most 1/4 of itself (1 to 1.5, in
    the middle of a step of 1/2) or 1/12 of the block's largest, an mxfp4 block's largest lies up to
    1/4 above 6; in a sum of many products these average to well under half of the result's size,
    which a wrong expert, permutation or scale does not meet."""
    T, d, F, E, k = 400, 512, 512, 8, 2
    x, mod, (w1, w3, w2) = _make(T, d, F, E, k, fmt)
    y, ids, w = mod(x, return_routing=True)
    want = torch.zeros(T, d, device="cuda")
    for j in range(k):
        for e in range(E):
            m = ids[:, j] == e
            xe = x[m].float()
            h = torch.nn.functional.silu(xe @ w1[e].T) * (xe @ w3[e].T)
            want[m] += (h @ w2[e].T) * w[m, j][:, None]
    assert (y.float() - want).norm() <= 0.5 * want.norm()


def test_layer_small_calls_and_host_buffers():
    x, mod, _ = _make(300, 256, 128, 8, 2, "nvfp4")
    assert mod(x[:0]).shape == (0, 256)
    y = mod(x)
    xh = x.cpu().pin_memory()
    yh = mod.forward_host(xh)
    torch.cuda.synchronize()
    assert torch.equal(yh, y.cpu())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yg = mod(x)
    x.copy_(x.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(yg, y.flip(0))        # every token's output depends on that token alone


def test_refusals_and_scales():
    x, mod, (w1, w3, w2) = _make(8, 64, 64, 4, 2, "mxfp4")
    with pytest.raises(ValueError):
        FP4MoELayer(mod.gate_weight, mod.experts, 2, input_scale=torch.ones(1))
    with pytest.raises(ValueError):
        FP4MoELayer(mod.gate_weight[:2], mod.experts, 2)
    with pytest.raises(ValueError):
        FP4Experts.from_dense(w1[:, :40], w3[:, :40], w2[:, :, :40])
    g = nvfp4_global_scale(torch.zeros(2, 3, 32, device="cuda"))
    assert torch.equal(g, torch.ones(2, device="cuda"))
    g = nvfp4_global_scale(torch.full((4, 32), -5.376, device="cuda"))
    assert g.shape == (1,) and abs(g.item() - 0.002) < 1e-9


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_no_experts(fmt):
    z = lambda *s: torch.empty(*s, device="cuda")
    ex = FP4Experts.from_dense(z(0, 64, 32), z(0, 64, 32), z(0, 32, 64), fmt)
    assert ex.num_experts == 0 and ex.w1[0].shape == (0, 64, 16) and ex.w2[0].shape == (0, 32, 32)


def test_new_scales_hold_from_the_next_call_on():
    """Values copied into the layer's scales, loaded or copied before a replay reach the quantisers and
    the products alike."""
    x, mod, _ = _make(37, 256, 96, 8, 2, "nvfp4", 1, 1, True)
    graph = torch.cuda.CUDAGraph()
    mod(x)
    with torch.cuda.graph(graph):
        yg = mod(x)
    for scale in (4.0, 0.25):
        mod.input_scale.fill_(0.002 * scale)
        mod.hidden_scale.mul_(scale)
        want = _by_hand(mod, x, 37, 2)[0]
        assert torch.equal(mod(x), want)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(yg, want)
    other = _make(37, 256, 96, 8, 2, "nvfp4", 1, 1, True)[1]
    saved = dict(mod.state_dict(), _alpha1=torch.ones(9), _alpha2=torch.ones(9), _alpha3=torch.ones(9))
    other.load_state_dict(saved)
    assert torch.equal(other(x), want)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32, torch.float64])
def test_casts_leave_the_scales_in_fp32(dt):
    x, mod, _ = _make(37, 256, 96, 8, 2, "nvfp4", 1, 1, True)
    y, scales = mod(x), (mod.input_scale.clone(), mod.hidden_scale.clone())
    mod.to(dt)
    assert mod.gate_weight.dtype == dt
    for a, b in zip((mod.input_scale, mod.hidden_scale), scales):
        assert a.dtype == torch.float32 and torch.equal(a, b)
    z = mod(x)
    assert z.shape == y.shape and z.dtype == y.dtype
    if dt == torch.bfloat16:
        assert torch.equal(z, y)
    mod.cpu()
    assert all(b.device.type == "cpu" for b in mod.buffers())
    assert mod.cuda().input_scale.device == x.device


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_ranges_of_a_host_batch_on_the_other_kernel(fmt):
    """1400 tokens are more rows than the products' rule gives to the kernel for few, a third of them
    are not: the ranges' results are the whole batch's, bit by bit."""
    x, mod, _ = _make(1400, 256, 96, 64, 2, fmt, S=1)
    xh = x.cpu().pin_memory()
    for chunks in (1, 2, 3):
        yh = mod.forward_host(xh, chunks=chunks)
        torch.cuda.synchronize()
        assert torch.equal(yh, mod(x).cpu())


def test_experts_of_parameters_keep_no_graph():
    """Quantised from trainable weights: scales without a history, which would hold the dense weights."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.nn.Parameter(torch.randn(*s, generator=gen, device="cuda"))
    w1, w3, w2, gate, scale = r(4, 96, 64), r(4, 96, 64), r(4, 64, 96), r(4, 64), r(1)
    ex = FP4Experts.from_dense(w1, w3, w2, "nvfp4", shared=[(r(96, 64), r(96, 64), r(64, 96))])
    assert not nvfp4_global_scale(w1).requires_grad
    assert not any(t.requires_grad for t in (ex.g1, ex.g3, ex.g2, *ex.w1, *ex.w3, *ex.w2))
    mod = FP4MoELayer(gate, ex, 2, gate_bias=r(4), input_scale=scale.abs(), hidden_scale=scale.abs())
    assert not any(b.requires_grad for b in mod.buffers())
    assert not mod(torch.randn(5, 64, device="cuda")).requires_grad
