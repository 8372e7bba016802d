"""GPU tests of the MoE layer for a few tokens against its definition in 64 bits.

The tolerance is derived from the layer's arithmetic.  Products of the operands are exact and summed in
fp32: at most 2^-23 of the sum of absolute values for each addition (the tensor core's may truncate).
Hidden values enter the second product as a sum of two 16-bit numbers: off by 2^-22 (fp16) or 2^-18
(bf16) of their value and 2^-39 of the largest; bf16 tokens as fp16 numbers lose 2^-39 of the largest.
The activation's exponential, division and products: 2^-20.  One rounding to the output type.  The
routing weights are checked by themselves, and the output is computed from the returned ones.
"""
import itertools

import numpy as np
import pytest
import torch

from light_moe_b200 import capi, ops

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
KINDS = [("fp8", "bf16"), ("fp8", "fp16"), ("dense", "bf16"), ("dense", "fp16")]


class Layer:
    def __init__(self, kind, d, F, E, k, S=0, bias=False, seed=0, std=0.05):
        weights, dt = kind
        self.dt, self.k, self.S, self.E, self.F = DT[dt], k, S, E, F
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=self.gen, device="cuda")
        self.gate = (r(E, d) / d ** 0.5).to(self.dt)
        self.bias = r(E) * 0.3 if bias else None
        self.scales = {}
        self.w = []
        for name, shape in (("w1", (E + S, F, d)), ("w3", (E + S, F, d)), ("w2", (E + S, d, F))):
            w = r(*shape) * std
            if weights == "fp8":
                q, s = ops.quantize_fp8(w, block_rows=128)
                s *= torch.exp2(torch.randint(-2, 3, s.shape, generator=self.gen, device="cuda").float())
                self.w.append(q)
                self.scales[name + "_scales"] = s
            else:
                self.w.append(w.to(self.dt))

    def x(self, T, outliers=True):
        x = torch.randn(T, self.gate.shape[1], generator=self.gen, device="cuda")
        if outliers:
            x[:, ::13] *= 30
        return x.to(self.dt)

    def __call__(self, x, **kw):
        return ops.moe_layer_few_tokens(x, self.gate, *self.w, self.k, num_shared=self.S, gate_bias=self.bias,
                                        **self.scales, **kw)

    def matrix(self, i, e):
        w = self.w[i][e].double()
        if self.scales:
            s = list(self.scales.values())[i][e].double()
            w = w * s.repeat_interleave(128, 0)[:w.shape[0]].repeat_interleave(128, 1)[:, :w.shape[1]]
        return w

    def logits(self, x):
        l = x.double() @ self.gate.double().T
        if self.bias is not None:
            l = l + self.bias.double()
        err = x.shape[1] * 2.0 ** -23 * (x.double().abs() @ self.gate.double().abs().T) + 2.0 ** -23 * l.abs()
        return l, err

    def check(self, x, out=None, exact_ids=True):
        y, ids, weights = out or self(x)
        T, d = x.shape
        assert y.shape == x.shape and y.dtype == x.dtype
        assert ids.shape == weights.shape == (T, self.k) and ids.dtype == torch.int32 and weights.dtype == torch.float32
        l, lerr = self.logits(x)
        order = torch.sort(l, dim=1, descending=True, stable=True)[1]
        chosen = torch.zeros(T, self.E, dtype=torch.bool, device="cuda").scatter_(1, ids.long(), True)
        assert (chosen.sum(1) == self.k).all()
        # logits that are left out are not larger than chosen ones, but for their errors; the order is descending
        low = torch.where(chosen, l + lerr, torch.full_like(l, float("inf"))).amin(1)
        high = torch.where(chosen, torch.full_like(l, -float("inf")), l - lerr).amax(1)
        assert (low >= high).all()
        got = l.gather(1, ids.long())
        tol = lerr.gather(1, ids.long())
        assert (got[:, :-1] + tol[:, :-1] >= got[:, 1:] - tol[:, 1:]).all()
        if exact_ids:
            sorted_l = l.gather(1, order)
            clear = (sorted_l[:, :-1] - sorted_l[:, 1:])[:, :self.k].amin(1) > 2 * lerr.amax(1) if self.E > 1 else \
                torch.ones(T, dtype=torch.bool, device="cuda")
            assert clear.double().mean() >= 0.5 and torch.equal(ids[clear].long(), order[clear][:, :self.k])
        want = torch.softmax(got, 1)
        # (an exponential below fp32's end, 2^-149, is 0)
        assert ((weights.double() - want).abs()
                <= want * (torch.expm1(2 * tol.amax(1, keepdim=True)) + 2.0 ** -20) + 2.0 ** -148).all()
        # the output, from the returned routing
        xd, top = x.double(), x.double().abs().amax(1, keepdim=True)
        want, err = torch.zeros(T, d, dtype=torch.float64, device="cuda"), torch.zeros(T, d, dtype=torch.float64, device="cuda")
        hs = []
        rel = d * 2.0 ** -23
        lost = top * 2.0 ** -39 if self.scales and self.dt == torch.bfloat16 else top * 0
        for e in range(self.E + self.S):
            if e < self.E:
                t = (ids == e).any(1).nonzero()[:, 0]
                w = (weights * (ids == e)).sum(1)[t][:, None].double()
            else:
                t = torch.arange(T, device="cuda")
                w = torch.ones(T, 1, dtype=torch.float64, device="cuda")
            if len(t) == 0:
                continue
            w1, w3, w2 = (self.matrix(i, e) for i in range(3))
            g, u = xd[t] @ w1.T, xd[t] @ w3.T
            dg = rel * (xd[t].abs() @ w1.abs().T) + lost[t] * w1.abs().sum(1)
            du = rel * (xd[t].abs() @ w3.abs().T) + lost[t] * w3.abs().sum(1)
            h = g * torch.sigmoid(g) * u * w
            # |silu'| <= 1.1
            dh = w * (1.1 * dg * (u.abs() + du) + g.abs() * torch.sigmoid(g) * du) + 2.0 ** -20 * h.abs()
            dh = dh + (2.0 ** -18 if not self.scales and self.dt == torch.bfloat16 else 2.0 ** -22) * h.abs()
            # fp32 ends at 2^-149: silu * up and its product with w are each off by 2^-150 there (tokens of 1e-30
            # have hidden values of 1e-60, which no fp32 number is near to)
            hs.append((t, h, dh + 2.0 ** -149, w2))
        hmax = torch.zeros(T, 1, dtype=torch.float64, device="cuda")
        for t, h, dh, w2 in hs:
            hmax[t] = torch.maximum(hmax[t], h.abs().amax(1, keepdim=True))
        n = len(hs) * self.F
        for t, h, dh, w2 in hs:
            want[t] += h @ w2.T
            err[t] += (dh + 2.0 ** -39 * hmax[t] + n * 2.0 ** -23 * h.abs()) @ w2.abs().T
        # the types end at 2^-24 and 2^-133: half of that
        bound = err + HALF[self.dt] * (want.abs() + err) + (2.0 ** -25 if self.dt == torch.float16 else 2.0 ** -134)
        bad = (y.double() - want).abs() > bound
        assert not bad.any(), (bad.nonzero()[:4].tolist(), bad.sum().item())
        return y


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [1, 2, 3, 8, 9, 16])
@pytest.mark.parametrize("d,F,E,k,S,bias", [
    (64, 32, 1, 1, 0, False), (128, 96, 4, 2, 1, True), (192, 160, 3, 3, 0, False), (320, 64, 40, 16, 3, False),
    (1024, 2816, 8, 2, 0, True), (4160, 224, 5, 2, 0, False)])
def test_layer(kind, T, d, F, E, k, S, bias):
    m = Layer(kind, d, F, E, k, S, bias, seed=T + d)
    m.check(m.x(T))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [1, 7, 16])
def test_layer_of_many_experts(kind, T):
    m = Layer(kind, 2048, 704, 64, 6, 2, seed=T)
    m.check(m.x(T))
    m = Layer(kind, 256, 64, 256, 8, 16, seed=T)
    m.check(m.x(T))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [9, 13, 16])
def test_layer_of_tokens_in_two_groups(kind, T):
    """Sixteen tokens of this size do not fit shared memory."""
    m = Layer(kind, 8192, 96, 4, 2, 1, seed=T, std=0.02)
    m.check(m.x(T))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [9, 16])
@pytest.mark.parametrize("E,k", [(17, 3), (130, 16)])
def test_layer_of_two_groups_and_shared_router_weights(kind, T, E, k):
    """Tokens in two groups, and experts enough for pairs of CTAs to share the router's weights.  (Most tokens have two
    logits closer than the bound of 8192 products: the choice is checked against the bound.)"""
    m = Layer(kind, 8192, 64, E, k, 2, bias=True, seed=T + E, std=0.02)
    m.check(m.x(T), exact_ids=False)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [4, 5, 8, 9, 16])
def test_layer_of_hidden_values_staged_in_chunks(kind, T):
    """A slice of the second kernel has up to 66 steps of 128 hidden values (132 of 64) of T tokens at 4 bytes, more
    than 128 KB, and its last step ends inside an expert's last 128."""
    m = Layer(kind, 8192, 4128, 8, 4, seed=T, std=0.02)
    # The logits' bound is 8192 * 2^-23 of the sum of absolute values, here about 8192 * 0.8 * (12 * 0.8 + 24) / 13 / 90
    # = 190, so 0.19 on either side, while five gaps of eight normal logits of size 8 are often smaller: too few tokens
    # have clear choices to demand half.  The choice is checked against the bound all the same.
    m.check(m.x(T), exact_ids=False)


@pytest.mark.parametrize("kind", KINDS)
def test_ties_go_to_the_lower_id(kind):
    m = Layer(kind, 128, 64, 12, 3)
    m.gate[5] = m.gate[2]
    m.gate[9] = m.gate[2]
    m.gate[11] = m.gate[2]
    x = (m.gate[2].float() * 20).to(m.dt).repeat(4, 1)
    y, ids, w = m(x)
    assert (ids == torch.tensor([2, 5, 9], device="cuda", dtype=torch.int32)).all()
    assert torch.allclose(w, torch.full_like(w, 1 / 3), rtol=2.0 ** -20)
    m.gate.zero_()
    y, ids, w = m(m.x(2))
    assert (ids == torch.tensor([0, 1, 2], device="cuda", dtype=torch.int32)).all()
    m.check(m.x(2), exact_ids=False)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_token_that_is_not_finite_spoils_only_itself(kind, bad):
    m = Layer(kind, 256, 160, 6, 2, 1)
    x = m.x(5)
    want = m(x)
    x2 = x.clone()
    x2[3, 7] = bad
    y, ids, w = m(x2)
    keep = [0, 1, 2, 4]
    assert torch.equal(y[keep], want[0][keep]) and torch.equal(ids[keep], want[1][keep])
    assert torch.equal(w[keep], want[2][keep])
    assert not torch.isfinite(y[3]).any()
    assert ((ids[3] >= 0) & (ids[3] < 6)).all() and len(set(ids[3].tolist())) == 2


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [2, 3, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_weights_that_are_not_finite_spoil_only_their_experts_tokens(kind, T, which, bad):
    """An infinite or NaN weight, or a block's scale (NaN where the quantiser met such a weight)."""
    m = Layer(kind, 256, 160, 6, 2, seed=T)
    x = m.x(T)
    want = m(x)
    hits = [(want[1] == e).any(1) for e in range(m.E)]
    e = next(i for i in range(m.E) if hits[i].any() and not hits[i].all())
    if m.scales:
        list(m.scales.values())[which][e, -1, -1] = bad
    else:
        m.w[which][e, -3, -5] = bad
    y, ids, w = m(x)
    assert torch.equal(ids, want[1]) and torch.equal(w, want[2])
    assert torch.equal(y[~hits[e]], want[0][~hits[e]])
    assert not torch.isfinite(y[hits[e]]).all(1).any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("E", [4, 40])
@pytest.mark.parametrize("T", [1, 5, 16])
def test_a_router_whose_bias_leaves_no_expert(kind, E, T):
    """A softmax over nothing but -inf, or with +inf, has no value; experts masked by -inf among others weigh nothing."""
    m = Layer(kind, 128, 64, E, 3, bias=True, seed=E + T)
    x = m.x(T)
    m.bias[1:] = -float("inf")
    y, ids, w = m(x)
    assert (ids[:, 0] == 0).all() and (w[:, 0] == 1).all() and (w[:, 1:] == 0).all()
    assert torch.isfinite(y).all()
    for value in (-float("inf"), float("inf")):
        m.bias.fill_(value)
        y, ids, w = m(x)
        assert torch.isnan(w).all() and torch.isnan(y).all()
        assert all(len(set(r)) == 3 and min(r) >= 0 and max(r) < E for r in ids.tolist())
    m.bias.zero_()
    m.bias[2] = float("inf")
    y, ids, w = m(x)
    assert (ids[:, 0] == 2).all() and torch.isnan(w).all() and torch.isnan(y).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e3, 1e25])
def test_values_of_other_sizes(kind, size):
    """Tokens and weights far from 1 (where the type holds them)."""
    if kind[1] == "fp16" and not 1e-4 < size < 1e4:
        size = 2.0 ** -6 if size < 1 else 2.0 ** 6
    m = Layer(kind, 256, 192, 4, 2, std=0.05 if size < 1 else 0.05 / size ** 0.5)
    m.gate = (m.gate.float() / max(size, 1e-3)).to(m.dt) if kind[1] == "bf16" else m.gate
    x = (m.x(6).float() * size).to(m.dt)
    out = m(x)
    fine = torch.isfinite(x).all(1)   # (fp16 ends at 65504: tokens beyond have no value to be near to)
    assert fine.any()
    m.check(x[fine], [o[fine] for o in out], exact_ids=False)


@pytest.mark.parametrize("kind", KINDS)
def test_zero_tokens_and_zero_weights(kind):
    m = Layer(kind, 128, 64, 4, 2, 1)
    x = m.x(3)
    x[1] = 0
    y = m.check(x, exact_ids=False)
    assert (y[1] == 0).all()
    y, ids, w = m(x[:0])
    assert y.shape == (0, 128) and ids.shape == (0, 2) and w.shape == (0, 2)


def test_tokens_do_not_depend_on_each_other():
    """A token's output is the same whatever tokens stand beside it (to the last bits of its sums)."""
    m = Layer(("fp8", "bf16"), 512, 320, 8, 2, 1, seed=3)
    x = m.x(16)
    y, ids, w = m(x)
    for t in (0, 7, 15):
        y1, ids1, w1 = m(x[t:t + 1])
        assert torch.equal(ids1[0], ids[t]) and torch.allclose(w1[0], w[t], rtol=1e-5)
        assert ((y1[0].float() - y[t].float()).abs() <= 2.0 ** -7 * y[t].float().abs() + 1e-4 * y[t].float().abs().max()).all()


def test_same_bits_every_time_and_on_two_streams():
    m = Layer(("fp8", "bf16"), 1024, 1408, 16, 4, 1, seed=4)
    x = m.x(8)
    want = m(x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(10):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(m(x))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_two_graphs_of_one_layer():
    """Captured calls keep their workspaces to themselves, and read the tokens of the moment."""
    m = Layer(("dense", "bf16"), 512, 608, 8, 2, seed=5)
    xs = [m.x(1), m.x(5)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x in xs:
            m(x)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(m(x))
        graphs.append(g)
    for round_ in range(3):
        for x in xs:
            x.copy_(m.x(x.shape[0]))
        torch.cuda.synchronize()
        for g in graphs:
            with torch.cuda.stream(torch.cuda.Stream()):
                g.replay()
        torch.cuda.synchronize()
        for x, o in zip(xs, outs):
            assert all(torch.equal(a, b) for a, b in zip(o, m(x)))
            m.check(x, o)


def test_views_and_strides():
    m = Layer(("fp8", "bf16"), 256, 160, 4, 2, seed=6)
    x = m.x(5)
    want = m(x)
    wide = torch.zeros(5, 300, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:259] = x
    assert torch.equal(m(wide[:, 3:259])[0], want[0])
    odd = torch.zeros(m.w[0].numel() + 16, dtype=torch.uint8, device="cuda")[16:].view(m.w[0].shape)
    odd.copy_(m.w[0].view(torch.uint8))
    m.w[0] = odd.view(torch.float8_e4m3fn)                      # 16-byte aligned only
    m.w[2] = m.w[2].view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(torch.float8_e4m3fn)
    m.scales["w3_scales"] = m.scales["w3_scales"].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(m(x)[0], want[0])


def _split_hidden_value():
    """Gate and up, integers of 12 bits, whose product h has a bf16 part, a rest with a bf16 part, and a rest of that
    of at least 2^-18 of h: (gate, up, first two parts, last part)."""
    b = lambda v: torch.tensor(float(v), dtype=torch.float64).to(torch.bfloat16).double().item()
    for g, u in itertools.product(range(2049, 2400, 2), range(2049, 2400, 2)):
        h = g * u
        parts = [b(h)]
        parts.append(b(h - parts[0]))
        last = h - parts[0] - parts[1]
        if abs(last) >= h * 2.0 ** -18 and parts[1] != 0:
            return g, u, parts, last
    raise AssertionError


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("F", [32, 4160])
def test_hidden_values_enter_the_second_product_with_all_bits(T, F, dt):
    """Three features that cancel but for the last 8 of 24 bits of the first.  The gates are large enough for
    silu(gate) = gate, and every number up to the second product is exact.  Two fp16 numbers lose at most 2^-22 of the value;
    the second product adds a handful of numbers of its size, each sum off by 2^-23 of it at most: 2^-20 together, where a second
    bf16 part's rest is 2^-18 or more."""
    g, u, parts, last = _split_hidden_value()
    d, t = 64, DT[dt]
    w1, w3 = (torch.zeros(1, F, d, device="cuda") for _ in range(2))
    w2 = torch.zeros(1, d, F, device="cuda")
    at = [1, F // 2, F - 1]
    # tokens are (1, 2^-8) times a power of two: a value of 12 bits is its high part + 256 * low part * 2^-8
    for w, v in ((w1, g), (w3, u)):
        w[0, at[0], 0], w[0, at[0], 1] = v // 16 * 16, (v % 16) * 256
    for i, p in zip(at[1:], parts):
        m, e = np.frexp(p)          # p = (m * 2^12) * 2^(e - 12): a gate of 2048 and more
        w1[0, i, 0], w3[0, i, 0] = abs(m) * 4096, np.sign(p) * 2.0 ** (int(e) - 12)
    w2[0, :, at[0]], w2[0, :, at[1]], w2[0, :, at[2]] = 1, -1, -1
    w = [v.to(t) for v in (w1, w3, w2)]
    assert all(torch.equal(a.float(), b) for a, b in zip(w, (w1, w3, w2)))
    s = torch.exp2((torch.arange(T, device="cuda") % 3).float() - 3)
    x = torch.zeros(T, d, device="cuda")
    x[:, 0], x[:, 1] = s, s * 2.0 ** -8
    y, _, _ = ops.moe_layer_few_tokens(x.to(t), torch.zeros(1, d, device="cuda", dtype=t), *w, 1)
    want = (last * s.double() ** 2)[:, None].expand(T, d)
    bound = 2.0 ** -20 * g * u * s.double()[:, None] ** 2 + HALF[t] * want.abs() * 1.01
    assert (bound < 0.5 * want.abs()).all()
    assert ((y.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("weights", ["fp8", "dense"])
def test_layer_of_more_than_2_to_the_31_weights(weights):
    """The last of several large experts is what it is as the only one."""
    d, F, E = 16384, 14336, 10
    m = Layer((weights, "bf16"), d, F, 1, 1, seed=9, std=0.02)
    x = m.x(2)
    want = m(x)
    for i in range(3):
        w = torch.zeros(E, *m.w[i].shape[1:], dtype=m.w[i].dtype, device="cuda")
        w[-1:] = m.w[i]
        m.w[i] = w
    assert m.w[0].numel() > 2 ** 31
    for name, s in m.scales.items():
        m.scales[name] = torch.cat([torch.ones_like(s)] * (E - 1) + [s])
    m.gate = torch.zeros(E, d, dtype=m.dt, device="cuda")
    m.bias = torch.zeros(E, device="cuda")
    m.bias[-1] = 1.0
    y, ids, w = m(x)
    assert (ids == E - 1).all() and (w == 1).all() and torch.equal(y, want[0])


def test_under_a_limit_of_ctas():
    m = Layer(("dense", "fp16"), 512, 608, 8, 2, seed=7)
    x = m.x(4)
    want = m(x)
    capi.lib().lmoe_set_gemm_sm_limit(3)
    try:
        got = m(x)
    finally:
        capi.lib().lmoe_set_gemm_sm_limit(0)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def _grids(call):
    """Grid sizes of the kernels that a captured call launches."""
    from cuda.bindings import driver
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    raw = driver.CUgraph(graph.raw_cuda_graph())
    ok = driver.CUresult.CUDA_SUCCESS
    err, _, n = driver.cuGraphGetNodes(raw)
    assert err == ok
    err, nodes, n = driver.cuGraphGetNodes(raw, n)
    assert err == ok
    sizes = []
    for node in nodes:
        err, kind = driver.cuGraphNodeGetType(node)
        assert err == ok
        if kind == driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            err, p = driver.cuGraphKernelNodeGetParams(node)
            assert err == ok
            sizes.append(p.gridDimX * p.gridDimY * p.gridDimZ)
    return sizes


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("limit", [1, 3, 32])
@pytest.mark.parametrize("T,d,E,S", [(1, 512, 8, 0), (4, 1024, 8, 1), (12, 512, 40, 2), (16, 8192, 4, 0)])
def test_both_kernels_keep_a_limit_of_ctas(kind, limit, T, d, E, S):
    m = Layer(kind, d, 608, E, 2, S, seed=T)
    x = m.x(T)
    want = m(x)
    assert max(_grids(lambda: m(x))) > 32
    capi.call("lmoe_set_gemm_sm_limit", limit)
    try:
        got = m(x)
        sizes = _grids(lambda: m(x))
    finally:
        capi.call("lmoe_set_gemm_sm_limit", 0)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert max(sizes) <= max(limit, 2)   # the first kernel's CTAs come in pairs


def test_refusals():
    m = Layer(("fp8", "bf16"), 128, 64, 4, 2)
    x = m.x(4)
    call = lambda x=x, gate=m.gate, w=m.w, k=2, sc=m.scales, **kw: ops.moe_layer_few_tokens(x, gate, *w, k, **sc, **kw)
    swapped = dict(m.scales, w1_scales=None)
    dense = [w.to(torch.float16) for w in m.w]
    for f, msg in (
            (lambda: call(m.x(17)), "at most 16"),
            (lambda: call(x.float()), "bf16 or fp16"),
            (lambda: call(x.half()), "differ in dtype"),
            (lambda: call(x[:, :64]), "gate_weight"),
            (lambda: call(x[0]), "x \\[T,d\\]"),
            (lambda: call(k=5), "top_k"),
            (lambda: call(k=0), "top_k"),
            (lambda: call(num_shared=1), "E\\+S"),
            (lambda: call(num_shared=-1), "num_shared"),
            (lambda: call(sc=swapped), "belong together"),
            (lambda: call(sc={}), "x's dtype"),
            (lambda: call(w=dense, sc={}), "x's dtype"),
            (lambda: call(w=dense), "float8_e4m3fn"),
            (lambda: call(w=[m.w[0], m.w[1][:, :32], m.w[2]]), "w1 and w3"),
            (lambda: call(sc=dict(m.scales, w2_scales=m.scales["w2_scales"].half())), "fp32"),
            (lambda: call(sc=dict(m.scales, w2_scales=m.scales["w2_scales"][:3])), "scales shape"),
            (lambda: call(gate_bias=torch.zeros(3, device="cuda")), "gate_bias"),
            (lambda: call(gate_bias=torch.zeros(4, device="cuda").half()), "gate_bias"),
            (lambda: call(gate=m.gate.cpu()), "CUDA"),
            (lambda: call(w=[m.w[0][:, :48], m.w[1][:, :48], m.w[2][:, :, :48]]), "multiple of 32")):
        with pytest.raises(RuntimeError, match=msg):
            f()
    big = Layer(("dense", "bf16"), 16384, 32, 1, 1)
    with pytest.raises(RuntimeError):   # eight tokens of this size do not fit shared memory
        big(big.x(8))
    big.check(big.x(2))
