"""GPU tests of the MoE layer with 8-bit experts: its steps together, against the steps called one by one,
and the few-token kernels against the kernels for larger batches."""
import pytest
import torch

from light_moe_b200 import ops
from light_moe_b200.fp8 import FEW_TOKENS, FP8Experts, FP8MoELayer

pytestmark = pytest.mark.gpu


def _make(T, d, F, E, k, S=0, seed=0, bias=False, power=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x = r(T, d).to(torch.bfloat16)
    w1, w3, w2 = r(E + S, F, d) * 0.05, r(E + S, F, d) * 0.05, r(E + S, d, F) * 0.05
    shared = [(w1[E + s], w3[E + s], w2[E + s]) for s in range(S)] or None
    ex = FP8Experts.from_dense(w1[:E], w3[:E], w2[:E], power, shared=shared)
    return x, FP8MoELayer(r(E, d) * 0.05, ex, k, gate_bias=r(E) * 0.1 if bias else None), (w1, w3, w2)


def _by_hand(mod, x, T, k):
    """The larger batches' steps without the permutation inside the quantiser: gather, then quantise."""
    e = mod.experts
    ids, w, _, off, sidx, pos = ops.fused_gate_topk_ex(x, mod.gate_weight, k, mod.gate_bias)[:6]
    rows = x[(sidx // k).long()]
    bounds = off
    if e.num_shared:
        rows = torch.cat([rows] + [x] * e.num_shared)
        bounds = torch.cat([off, off[-1:] + T * torch.arange(1, e.num_shared + 1, device="cuda", dtype=torch.int32)])
    n = e.num_experts + e.num_shared
    h = ops.fp8_grouped_gemm(*ops.quantize_fp8(rows), *e.w1, bounds, n, weights_up=e.w3[0], weight_scales_up=e.w3[1])
    o = ops.fp8_grouped_gemm(*ops.quantize_fp8(h), *e.w2, bounds, n)
    y = torch.zeros(T, x.shape[1], device="cuda")
    for j in range(k):
        y = y + w[:, j:j + 1] * o[pos.view(T, k)[:, j].long()].float()
    for s in range(e.num_shared):
        y = y + o[T * k + s * T:T * k + (s + 1) * T].float()
    return y.to(torch.bfloat16), ids, w


@pytest.mark.parametrize("power", [False, True])
@pytest.mark.parametrize("T,d,F,E,k,S,bias", [(FEW_TOKENS + 1, 256, 128, 8, 2, 0, False), (37, 256, 96, 8, 2, 0, True),
                                              (300, 128, 144, 16, 4, 2, False), (1500, 256, 256, 4, 2, 1, True)])
def test_layer_equals_its_steps(T, d, F, E, k, S, bias, power):
    x, mod, _ = _make(T, d, F, E, k, S, T, bias, power)
    y, ids, w = mod(x, return_routing=True)
    want, ids2, w2 = _by_hand(mod, x, T, k)
    assert torch.equal(ids, ids2) and torch.equal(w, w2)
    assert torch.equal(y, want)
    assert torch.equal(mod(x.view(1, T, d)).view(T, d), y)


@pytest.mark.parametrize("T", [FEW_TOKENS + 1, 300])
@pytest.mark.parametrize("S", [1, 3])
def test_layer_of_256_experts_and_shared_ones(T, S):
    """More experts than one product takes: routed and shared ones by themselves, for a few tokens together."""
    x, mod, _ = _make(T, 64, 32, 256, 8, S, seed=T, bias=True)
    y, ids, w = mod(x, return_routing=True)
    e, k = mod.experts, 8
    ids2, w2, _, off, sidx, pos = ops.fused_gate_topk_ex(x, mod.gate_weight, k, mod.gate_bias)[:6]
    assert torch.equal(ids, ids2) and torch.equal(w, w2)

    def run(rows, offsets, a, b):
        part = lambda m: (m[0][a:b], m[1][a:b])
        h = ops.fp8_grouped_gemm(*ops.quantize_fp8(rows), *part(e.w1), offsets, b - a, weights_up=e.w3[0][a:b],
                                 weight_scales_up=e.w3[1][a:b])
        return ops.fp8_grouped_gemm(*ops.quantize_fp8(h), *part(e.w2), offsets, b - a)

    o = run(x[(sidx // k).long()], off, 0, 256)
    want = torch.zeros(T, 64, device="cuda")
    for j in range(k):
        want = want + w[:, j:j + 1] * o[pos.view(T, k)[:, j].long()].float()
    for s in range(S):
        want = want + run(x, torch.tensor([0, T], dtype=torch.int32, device="cuda"), 256 + s, 257 + s).float()
    assert torch.equal(y, want.to(torch.bfloat16))
    few, ids, w = mod(x[:5], return_routing=True)
    assert torch.equal(ids, ids2[:5]) and torch.allclose(w, w2[:5], rtol=1e-4)
    assert (few.float() - y[:5].float()).norm() <= 2.0 ** -4 * few.float().norm()   # (E4M3 activations, as above)


def test_layers_that_no_call_could_run_are_refused():
    x, mod, (w1, w3, w2) = _make(1, 64, 32, 4, 2, 1)
    many = lambda n: FP8Experts(*((q[:1].expand(n, -1, -1), s[:1].expand(n, -1, -1)) for q, s in
                                  (mod.experts.w1, mod.experts.w3, mod.experts.w2)), n, 0, 64, 32)
    for experts, k in ((many(257), 2), (mod.experts, 0), (mod.experts, 5), (many(40), 17)):
        with pytest.raises(ValueError):
            FP8MoELayer(torch.zeros(experts.num_experts, 64, device="cuda"), experts, k)
    shared = FP8Experts(*((q[:1].expand(258, -1, -1), s[:1].expand(258, -1, -1)) for q, s in
                          (mod.experts.w1, mod.experts.w3, mod.experts.w2)), 1, 257, 64, 32)
    with pytest.raises(ValueError):
        FP8MoELayer(torch.zeros(1, 64, device="cuda"), shared, 1)


def test_ffn_sizes_beyond_the_few_token_kernels():
    """They run like larger batches, row by row the same."""
    x, mod, _ = _make(FEW_TOKENS + 1, 64, 65568, 1, 1)
    y = mod(x)
    for T in (1, 5):
        assert torch.equal(mod(x[:T]), y[:T])


@pytest.mark.parametrize("T", [1, 5, FEW_TOKENS])
def test_few_tokens_take_their_kernels(T):
    x, mod, _ = _make(T, 256, 96, 8, 2, 1, T, True)
    e = mod.experts
    y, ids, w = mod(x, return_routing=True)
    want = ops.moe_layer_few_tokens(x, mod.gate_weight, e.w1[0], e.w3[0], e.w2[0], 2, e.w1[1], e.w3[1], e.w2[1], 1,
                                    mod.gate_bias)
    assert all(torch.equal(a, b) for a, b in zip((y, ids, w), want))
    # the other kernels quantise tokens and hidden values: E4M3 is off by 2^-4 at most, 2^-4 / sqrt(3) rms at the worst place
    # of a step and less elsewhere; both stages together stay below 2^-4 of a sum of many products
    other, ids2, w2 = _by_hand(mod, x, T, 2)
    assert torch.equal(ids, ids2) and torch.allclose(w, w2, rtol=1e-4)
    assert (y.float() - other.float()).norm() <= 2.0 ** -4 * y.float().norm()


@pytest.mark.parametrize("T", [9, 400])
def test_layer_is_near_the_dense_experts(T):
    """E4M3 values are off by 2^-4 of themselves at most; weights, tokens and hidden values together, in sums of
    many products, by far less than 1/8, which a wrong expert, permutation or scale does not meet."""
    d, F, E, k = 512, 512, 8, 2
    x, mod, (w1, w3, w2) = _make(T, d, F, E, k)
    y, ids, w = mod(x, return_routing=True)
    want = torch.zeros(T, d, device="cuda")
    for j in range(k):
        for e in range(E):
            m = ids[:, j] == e
            xe = x[m].float()
            h = torch.nn.functional.silu(xe @ w1[e].T) * (xe @ w3[e].T)
            want[m] += (h @ w2[e].T) * w[m, j][:, None]
    assert (y.float() - want).norm() <= 0.125 * want.norm()


@pytest.mark.parametrize("T", [7, 300])
def test_layer_small_calls_and_host_buffers(T):
    x, mod, _ = _make(T, 256, 128, 8, 2)
    assert mod(x[:0]).shape == (0, 256)
    y, ids, w = mod(x[:0], return_routing=True)
    assert ids.shape == w.shape == (0, 2)
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
    assert torch.equal(yg, mod(x))
    if T > FEW_TOKENS:
        assert torch.equal(yg, y.flip(0))        # every token's output depends on that token alone


def test_ranges_of_a_host_batch():
    x, mod, _ = _make(1400, 256, 96, 64, 2, 1)
    xh = x.cpu().pin_memory()
    for chunks in (1, 2, 3, 10):
        yh = mod.forward_host(xh, chunks=chunks)
        torch.cuda.synchronize()
        assert torch.equal(yh, mod(x).cpu())


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32, torch.float64])
@pytest.mark.parametrize("T", [3, 37])
def test_casts_of_the_module(T, dt):
    x, mod, _ = _make(T, 256, 96, 8, 2, 1, 1, True)
    y = mod(x)
    mod.to(dt)
    assert mod.gate_weight.dtype == dt
    z = mod(x)
    assert z.shape == y.shape and z.dtype == y.dtype
    if dt == torch.float32 and T <= FEW_TOKENS:
        assert torch.equal(z, y)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32, torch.float64])
@pytest.mark.parametrize("T", [3, 37])
def test_casts_of_the_module_keep_its_values(T, dt):
    """A cast layer computes what its cast router says: a few tokens what a layer built from it computes, more tokens what
    the steps called one by one do; and its routing is near the softmax in 64 bits."""
    x, mod, _ = _make(T, 256, 96, 8, 2, 1, 1, True)
    mod.to(dt)
    gate, bias = mod.gate_weight, mod.gate_bias
    y, ids, w = mod(x, return_routing=True)
    if T <= FEW_TOKENS:
        want, ids2, w2 = FP8MoELayer(gate, mod.experts, 2, bias)(x, return_routing=True)
    else:
        want, ids2, w2 = _by_hand(mod, x, T, 2)
    assert torch.equal(y, want) and torch.equal(ids, ids2) and torch.equal(w, w2)
    # 256 products and the bias in fp32, each sum off by 2^-23 of the sum of absolute values at most
    l = x.double() @ gate.double().T + bias.double()
    err = 257 * 2.0 ** -23 * (x.double().abs() @ gate.double().abs().T + bias.double().abs())
    chosen = torch.zeros_like(l, dtype=torch.bool).scatter_(1, ids.long(), True)
    assert (chosen.sum(1) == 2).all()
    assert ((l + err)[chosen].view(T, 2).amin(1) >= (l - err).masked_fill(chosen, -float("inf")).amax(1)).all()
    want = torch.softmax(l.gather(1, ids.long()), 1)
    # the exponentials' errors, 2 units in the last place, the sum and the quotient: 2^-20
    assert ((w.double() - want).abs() <= want * (torch.expm1(2 * err.amax(1, keepdim=True)) + 2.0 ** -20)).all()


def test_experts_of_a_checkpoint():
    x, mod, _ = _make(20, 128, 208, 4, 2, 1)
    e = mod.experts
    strided = lambda w: (w[0], w[1].transpose(1, 2).contiguous().transpose(1, 2))
    again = FP8MoELayer(mod.gate_weight, FP8Experts.from_quantized(strided(e.w1), strided(e.w3), strided(e.w2), 4), 2)
    assert again.experts.num_shared == 1 and torch.equal(again(x), mod(x))
    assert torch.equal(again(x[:3]), mod(x[:3]))


def test_experts_of_parameters_keep_no_graph():
    gen = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.nn.Parameter(torch.randn(*s, generator=gen, device="cuda"))
    ex = FP8Experts.from_dense(r(4, 96, 64), r(4, 96, 64), r(4, 64, 96), shared=[(r(96, 64), r(96, 64), r(64, 96))])
    assert not any(t.requires_grad for t in (*ex.w1, *ex.w3, *ex.w2))
    mod = FP8MoELayer(r(4, 64), ex, 2, gate_bias=r(4))
    assert not any(b.requires_grad for b in mod.buffers())
    x = torch.randn(40, 64, device="cuda", requires_grad=True)
    assert not mod(x[:5]).requires_grad and not mod(x).requires_grad


def test_refusals():
    x, mod, (w1, w3, w2) = _make(8, 64, 64, 4, 2)
    e = mod.experts
    with pytest.raises(ValueError):
        FP8MoELayer(mod.gate_weight[:2], e, 2)
    with pytest.raises(ValueError):
        FP8MoELayer(mod.gate_weight, e, 2, gate_bias=torch.zeros(3, device="cuda"))
    with pytest.raises(ValueError):
        FP8Experts.from_dense(w1[:, :40], w3[:, :40], w2[:, :, :48])
    with pytest.raises(RuntimeError):
        FP8Experts.from_dense(w1[:, :40], w3[:, :40], w2[:, :, :40])
    with pytest.raises(ValueError):
        FP8Experts.from_quantized(e.w1, e.w3, (e.w2[0], e.w2[1].half()), 4)
    with pytest.raises(ValueError):
        FP8Experts.from_quantized(e.w1, e.w3, (e.w2[0], e.w2[1][:, :0]), 4)
    with pytest.raises(ValueError):
        FP8Experts.from_quantized(e.w1, e.w3, e.w2, 5)
    small = FP8Experts.from_dense(w1[:, :, :48], w3[:, :, :48], w2[:, :48])
    with pytest.raises(ValueError):   # the router wants multiples of 64
        FP8MoELayer(mod.gate_weight[:, :48], small, 2)
