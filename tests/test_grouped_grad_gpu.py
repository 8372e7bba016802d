"""GPU tests of the grouped product's gradients against the formula in 64 bits.

Tolerance, derived: 16-bit products are exact in fp32; L of them are summed in fp32, each addition
off by at most one unit in the last place (L * 2^-23 of the sum of absolute products); fp32
operands round each product once more inside the fused multiply-add (the same bound); the output
type rounds by eps / 2.
"""
import pytest
import torch

from light_moe_b200 import capi, ops

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _bounds(counts, head=0):
    b = [head]
    for c in counts:
        b.append(b[-1] + c)
    return b


def _inputs(counts, N, K, dt, head=0, tail=0, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    b = _bounds(counts, head)
    R, E = b[-1] + tail, len(counts)
    dy = torch.randn(R, N, generator=gen, device="cuda").to(dt)
    x = torch.randn(R, K, generator=gen, device="cuda").to(dt)
    w = (torch.randn(E, N, K, generator=gen, device="cuda") * 0.1).to(dt)
    return dy, x, w, b, torch.tensor(b, dtype=torch.int32, device="cuda")


def _close(got, want, mass, depth, what):
    half = torch.finfo(got.dtype).eps / 2
    tol = (depth + 1) * 2.0 ** -23 * mass * (1 + half) + half * want.abs() + torch.finfo(got.dtype).tiny
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (what, bad.sum().item(), (got.double() - want).abs().max().item())


def _check(dy, x, w, b, off, out_dtype=None):
    E = len(b) - 1
    dx = ops.grouped_gemm_dgrad(dy, w, off, E)
    dw = ops.grouped_gemm_wgrad(dy, x, off, E, out_dtype)
    assert dx.dtype == dy.dtype and dx.shape == x.shape
    assert dw.dtype == (out_dtype or dy.dtype) and dw.shape == w.shape
    assert (dx[:b[0]] == 0).all() and (dx[b[-1]:] == 0).all()
    for e in range(E):
        r = slice(b[e], b[e + 1])
        g, xe, we = dy[r].double(), x[r].double(), w[e].double()
        _close(dx[r], g @ we, g.abs() @ we.abs(), w.shape[1], f"dx {e}")
        _close(dw[e], g.T @ xe, g.abs().T @ xe.abs(), max(b[e + 1] - b[e], 1), f"dw {e}")
    return dx, dw


SHAPES = [
    ([1], 64, 64), ([1, 0, 3], 8, 16), ([256], 256, 256), ([64, 65, 15, 0, 17], 256, 512), ([130, 1, 300], 320, 264),
    ([5, 700], 1408, 520), ([33, 31], 72, 2048), ([2, 500, 2], 1000, 8),
]


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("counts,N,K", SHAPES)
def test_gradients(dt, counts, N, K):
    _check(*_inputs(counts, N, K, DT[dt], seed=N + K))


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("counts,N,K", [([3, 40], 1, 1), ([20, 0, 9], 33, 64), ([129, 60], 64, 129), ([70, 300], 257, 517),
                                        ([1], 7, 3)])
def test_gradients_of_odd_sizes(dt, counts, N, K):
    _check(*_inputs(counts, N, K, DT[dt], seed=N))


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("head,tail", [(0, 0), (7, 0), (0, 300), (290, 5)])
def test_rows_outside_every_expert(dt, head, tail):
    """Rows outside the experts hold NaN and infinities; neither gradient sees them."""
    dy, x, w, b, off = _inputs([30, 0, 100, 45], 136, 200, DT[dt], head, tail)
    for t in (dy, x):
        t[:b[0]] = float("nan")
        t[b[-1]:] = float("inf")
    _check(dy, x, w, b, off.long())


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_what_is_not_finite_stays_in_its_expert(dt):
    dy, x, w, b, off = _inputs([21, 50, 9, 70], 136, 136, DT[dt])
    dx0, dw0 = _check(dy, x, w, b, off)
    dy[b[1]] = float("nan")        # the row right behind expert 0
    x[b[2] - 1] = float("inf")     # the last row of expert 1
    w[2] = float("nan")            # right behind expert 1's matrix
    dx = ops.grouped_gemm_dgrad(dy, w, off, 4)
    dw = ops.grouped_gemm_wgrad(dy, x, off, 4)
    for e in (0, 3):
        assert torch.equal(dx[b[e]:b[e + 1]], dx0[b[e]:b[e + 1]]) and torch.equal(dw[e], dw0[e])
    assert torch.equal(dw[2], dw0[2])
    assert torch.isnan(dx[b[1]]).all() and torch.equal(dx[b[1] + 1:b[2]], dx0[b[1] + 1:b[2]])
    assert torch.isnan(dw[1]).all() and torch.isnan(dx[b[2]:b[3]]).all()


def test_weight_gradient_in_fp32_and_no_rows():
    for dt in (torch.bfloat16, torch.float16):
        _check(*_inputs([100, 0, 37], 264, 130, dt), out_dtype=torch.float32)
    dy, x, w, b, off = _inputs([0, 0], 64, 64, torch.bfloat16)
    assert ops.grouped_gemm_dgrad(dy, w, off, 2).shape == (0, 64)
    assert (ops.grouped_gemm_wgrad(dy, x, off, 2) == 0).all()
    assert (ops.grouped_gemm_wgrad(dy.float(), x.float(), off, 2) == 0).all()


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_many_experts(dt):
    _check(*_inputs([i % 5 * 9 for i in range(256)], 72, 80, DT[dt]))


def test_uneven_prompt():
    """Many tiles per pair of CTAs, loads from none to most of the rows."""
    _check(*_inputs([0, 3000, 41, 0, 640, 257, 1], 1408, 1024, torch.bfloat16))


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("offsets", [[0, 50, 40, 100], [-1, 20, 40, 100], [0, 20, 40, 101], [120, 130, 140, 150]])
def test_bad_offsets_give_zeros_and_an_error_word(dt, offsets):
    R, N, K, t = 100, 64, 64, DT[dt]
    code = capi.dtype_code(t)
    dy, x, w = (torch.ones(*s, device="cuda", dtype=t) for s in ((R, N), (R, K), (3, N, K)))
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    dx, dw = torch.full((R, K), 5.0, device="cuda", dtype=t), torch.full((3, N, K), 5.0, device="cuda", dtype=t)
    e1, e2 = (torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2))
    capi.call("lmoe_grouped_gemm_dgrad", dy.data_ptr(), code, R, N, w.data_ptr(), K, off.data_ptr(), 0, 3,
              dx.data_ptr(), None, 0, e1.data_ptr(), capi.stream_handle())
    capi.call("lmoe_grouped_gemm_wgrad", dy.data_ptr(), code, R, N, x.data_ptr(), K, off.data_ptr(), 0, 3, code,
              dw.data_ptr(), None, 0, e2.data_ptr(), capi.stream_handle())
    assert (dx == 0).all() and (dw == 0).all() and e1.item() != 0 and e2.item() != 0


def test_views_strides_and_more_weights_than_experts():
    dy, x, w, b, off = _inputs([40, 60], 64, 96, torch.bfloat16)
    dx, dw = _check(dy, x, w, b, off)
    wide = torch.zeros(100, 67, device="cuda", dtype=torch.bfloat16)
    wide[:, 3:] = dy
    assert torch.equal(ops.grouped_gemm_dgrad(wide[:, 3:], w, off, 2), dx)
    flat = torch.zeros(100 * 96 + 1, device="cuda", dtype=torch.bfloat16)
    flat[1:] = x.reshape(-1)
    assert torch.equal(ops.grouped_gemm_wgrad(dy, flat[1:].view(100, 96), off, 2), dw)   # contiguous, not aligned
    assert torch.equal(ops.grouped_gemm_wgrad(dy.t().contiguous().t(), x, off, 2), dw)
    more = torch.cat([w, torch.full_like(w, float("nan"))])
    assert torch.equal(ops.grouped_gemm_dgrad(dy, more, off, 2), dx)
    row = torch.randn(1, 64, device="cuda", dtype=torch.bfloat16).expand(100, 64)        # a broadcast gradient
    assert torch.equal(ops.grouped_gemm_dgrad(row, w, off, 2), ops.grouped_gemm_dgrad(row.contiguous(), w, off, 2))


def test_refusals_on_the_device():
    dy, x, w, b, off = _inputs([40, 60], 64, 96, torch.bfloat16)
    for call in (
        lambda: ops.grouped_gemm_dgrad(dy, w.float(), off, 2),
        lambda: ops.grouped_gemm_dgrad(dy[0], w, off, 2),
        lambda: ops.grouped_gemm_dgrad(dy[:, :32], w, off, 2),
        lambda: ops.grouped_gemm_dgrad(dy, w, off, 3),
        lambda: ops.grouped_gemm_dgrad(dy, w, off[:2], 2),
        lambda: ops.grouped_gemm_dgrad(dy, w, off.float(), 2),
        lambda: ops.grouped_gemm_dgrad(dy, w, off.cpu(), 2),
        lambda: ops.grouped_gemm_dgrad(dy, w.cpu(), off, 2),
        lambda: ops.grouped_gemm_dgrad(dy.double(), w.double(), off, 2),
        lambda: ops.grouped_gemm_wgrad(dy, x[:50], off, 2),
        lambda: ops.grouped_gemm_wgrad(dy, x.half(), off, 2),
        lambda: ops.grouped_gemm_wgrad(dy, x, off, 2, torch.float16),
        lambda: ops.grouped_gemm_wgrad(dy, x, off, 0),
    ):
        with pytest.raises(RuntimeError):
            call()


def test_streams_and_graphs():
    dy, x, w, b, off = _inputs([140, 0, 161], 264, 200, torch.bfloat16)
    dx, dw = _check(dy, x, w, b, off)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s1):
        a = ops.grouped_gemm_dgrad(dy, w, off, 3)
    with torch.cuda.stream(s2):
        c = ops.grouped_gemm_wgrad(dy, x, off, 3)
    torch.cuda.synchronize()
    assert torch.equal(a, dx) and torch.equal(c, dw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gx, gw = ops.grouped_gemm_dgrad(dy, w, off, 3), ops.grouped_gemm_wgrad(dy, x, off, 3)
    dy.copy_(dy.flip(0))
    off.copy_(torch.tensor([0, 10, 200, 301], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(gx, ops.grouped_gemm_dgrad(dy, w, off, 3))
    assert torch.equal(gw, ops.grouped_gemm_wgrad(dy, x, off, 3))


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("counts,N,K,head,tail", [([5], 7680, 856, 0, 0), ([3, 0, 2], 4099, 130, 2, 9), ([1], 1025, 1, 0, 3),
                                                  ([200, 90], 2048, 264, 1, 0)])
def test_long_contractions_of_few_tiles(dt, counts, N, K, head, tail):
    """The contraction is summed in ranges that are joined in order: the formula's values, the same
    bits in every run, and, without a workspace for the ranges, one sum."""
    dy, x, w, b, off = _inputs(counts, N, K, DT[dt], head, tail, seed=N)
    dx, _ = _check(dy, x, w, b, off)
    assert torch.equal(dx, ops.grouped_gemm_dgrad(dy, w, off, len(counts)))
    y = ops.grouped_gemm(dy, w.transpose(1, 2).contiguous(), off, len(counts))   # the same sums, K-major
    assert (y[:head] == 0).all() and (y[b[-1]:] == 0).all()
    for e in range(len(counts)):
        r = slice(b[e], b[e + 1])
        g, we = dy[r].double(), w[e].double()
        _close(y[r], g @ we, g.abs() @ we.abs(), N, f"product {e}")
    if N % 8 == 0 and K % 8 == 0:
        one = torch.empty_like(dx)
        capi.call("lmoe_grouped_gemm_dgrad", dy.data_ptr(), 0 if dt == "bf16" else 1, dy.shape[0], N, w.data_ptr(), K,
                  off.data_ptr(), 0, len(counts), one.data_ptr(), None, 0, None, capi.stream_handle())
        e = b[-1] - 1
        _close(one[e:e + 1], dy[e:e + 1].double() @ w[-1].double(), dy[e:e + 1].double().abs() @ w[-1].double().abs(), N, "one sum")


def test_fp32_of_every_magnitude():
    """fp32 operands near the largest value (whose high plane would round to an infinity) and tiny ones
    (whose lower planes end at 2^-133: half of that, 2^-134, is lost of each value) on tensor cores."""
    counts, N, K = [70, 33], 256, 200
    dy, x, w, b, off = _inputs(counts, N, K, torch.float32, seed=5)
    for scale, other in ((2.0 ** 126, 2.0 ** -60), (2.0 ** -115, 2.0 ** 40), (2.0 ** -124, 2.0 ** 30), (2.0 ** 60, 2.0 ** -100)):
        d, v, u = (dy.clamp(-3.9, 3.9) * scale), w * other, x * other
        dx, dw = ops.grouped_gemm_dgrad(d, v, off, 2), ops.grouped_gemm_wgrad(d, u, off, 2)
        lost = 2.0 ** -134
        for e in range(2):
            r = slice(b[e], b[e + 1])
            for got, p, q, depth in ((dx[r], d[r].double(), v[e].double(), N),
                                     (dw[e], d[r].double().T, u[r].double(), counts[e])):
                tol = (depth + 1) * 2.0 ** -23 * (p.abs() @ q.abs()) + 2.0 ** -148
                tol = tol + lost * (q.abs().sum(0)[None] + p.abs().sum(1)[:, None])
                assert torch.isfinite(got).all() and ((got.double() - p @ q).abs() <= tol).all(), (scale, other, e)


@pytest.mark.parametrize("dt,counts,N,K", [("fp32", [140, 0, 161], 264, 200), ("bf16", [5, 3], 4096, 256),
                                           ("fp16", [90, 41], 131, 77), ("fp32", [3, 2], 40, 24)])
def test_calls_at_once_and_replayed(dt, counts, N, K):
    """Two streams with calls in flight together, each with its workspaces; a captured pair replayed with
    other rows."""
    E = len(counts)
    dy, x, w, b, off = _inputs(counts, N, K, DT[dt])
    other = dy.flip(0).contiguous()
    want = [(ops.grouped_gemm_dgrad(g, w, off, E), ops.grouped_gemm_wgrad(g, x, off, E)) for g in (dy, other)]
    torch.cuda.synchronize()
    got = [[], []]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(8):
        for i, g in enumerate((dy, other)):
            with torch.cuda.stream(streams[i]):
                got[i].append((ops.grouped_gemm_dgrad(g, w, off, E), ops.grouped_gemm_wgrad(g, x, off, E)))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, want[i][0]) and torch.equal(c, want[i][1]) for a, c in got[i])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gx, gw = ops.grouped_gemm_dgrad(dy, w, off, E), ops.grouped_gemm_wgrad(dy, x, off, E)
    dy.copy_(other)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(gx, want[1][0]) and torch.equal(gw, want[1][1])


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("offsets", [[0, 50, 40, 100], [0, 20, 40, 101], [0, 50, 60, 100]])
def test_error_words_of_the_operators(dt, offsets):
    """Bad offsets set the caller's word and good ones leave it; fp32 sizes for CUDA cores and for planes."""
    bad = offsets != [0, 50, 60, 100]
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    for N, K in ((64, 64), (2048, 2880)):
        dy, x, w = (torch.ones(*s, device="cuda", dtype=DT[dt]) for s in ((100, N), (100, K), (3, N, K)))
        for call in (lambda e: ops.grouped_gemm_dgrad(dy, w, off, 3, error=e),
                     lambda e: ops.grouped_gemm_wgrad(dy, x, off, 3, error=e)):
            e = torch.zeros(1, dtype=torch.int32, device="cuda")
            y = call(e)
            assert (e.item() != 0) == bad and (y != 0).any().item() != bad
    for e in (torch.zeros(1, device="cuda"), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32, device="cuda")):
        with pytest.raises(RuntimeError):
            ops.grouped_gemm_dgrad(dy, w, off, 3, error=e)
        with pytest.raises(RuntimeError):
            ops.grouped_gemm_wgrad(dy, x, off, 3, error=e)


def test_error_words_name_the_kernel():
    """The low 24 bits of a word tell where it was set: another place for each kernel."""
    off = torch.tensor([0, 60, 40], dtype=torch.int32, device="cuda")
    sites = set()
    for dt, n in ((torch.bfloat16, 64), (torch.float32, 64), (torch.float32, 128)):   # 16-bit, CUDA cores, planes
        planes = capi.lib().lmoe_grouped_gemm_grad_workspace_bytes(0, capi.dtype_code(dt), 50, n, 64, 2) > 0
        assert planes == (n == 128)
        e = torch.zeros(1, dtype=torch.int32, device="cuda")
        ops.grouped_gemm_dgrad(torch.ones(50, n, device="cuda", dtype=dt), torch.ones(2, n, 64, device="cuda", dtype=dt),
                               off, 2, error=e)
        assert e.item() >> 24 == 2   # an argument outside its range
        sites.add(e.item() & 0xffffff)
    assert len(sites) == 3


# ------------------------------------------------------------------- fp32 as three bf16 planes
def _on_planes(form, R, N, K, E):
    """Whether a call of fp32 operands takes the kernel that splits them into planes."""
    return capi.lib().lmoe_grouped_gemm_grad_workspace_bytes(form, capi.LMOE_DTYPE_F32, R, N, K, E) > 0


def _one_per_column(shape, place, gen):
    """Random values at [.., place[c], c] and zeros elsewhere."""
    w = torch.zeros(shape, device="cuda")
    c = torch.arange(shape[-1], device="cuda")
    w[..., place, c] = torch.randn(*shape[:-2], shape[-1], generator=gen, device="cuda")
    return w


def test_planes_hold_every_bit():
    """One product x * y in each output: its error is that of the planes alone.  x = h + m + l exactly
    (8 bits each), |m| <= 2^-8 |x| and |l| <= 2^-16 |x|; the products (m, l), (l, m) and (l, l) are left
    out, 2^-23 |x y|; five additions of the other six are off by a unit in the last place, 2^-23 of at
    most (1 + 2^-7) |x y| each.  Together below 7 * 2^-23; without a plane it would be 2^-17 or more."""
    gen = torch.Generator(device="cuda").manual_seed(11)
    near = lambda got, want: ((got.double() - want).abs() <= 7 * 2.0 ** -23 * want.abs()).all()
    counts = [1, 70, 0, 33]
    b = _bounds(counts)
    off = torch.tensor(b, dtype=torch.int32, device="cuda")
    R, N, K = b[-1], 161, 200
    dy = torch.randn(R, N, generator=gen, device="cuda")
    assert _on_planes(0, R, N, K, 4)
    place = torch.arange(K, device="cuda") * 7 % N
    w = _one_per_column((4, N, K), place, gen)
    dx = ops.grouped_gemm_dgrad(dy, w, off, 4)
    assert _on_planes(2, R, K, N, 4)
    y = ops.grouped_gemm(dy, w.transpose(1, 2).contiguous(), off, 4)   # the same sums as a product of 161 values
    for e in range(4):
        r = slice(b[e], b[e + 1])
        want = dy[r][:, place].double() * w[e].sum(0).double()
        assert near(dx[r], want) and near(y[r], want)
    counts = [1, 70, 3, 130]
    b = _bounds(counts)
    off = torch.tensor(b, dtype=torch.int32, device="cuda")
    R, N, K = b[-1], 2048, 2056
    assert _on_planes(1, R, N, K, 4)
    dy, x = torch.randn(R, N, generator=gen, device="cuda"), torch.zeros(R, K, device="cuda")
    for e in range(4):
        x[b[e]:b[e + 1]] = _one_per_column((counts[e], K), torch.arange(K, device="cuda") * 3 % counts[e], gen)
    dw = ops.grouped_gemm_wgrad(dy, x, off, 4)
    for e in range(4):
        r = slice(b[e], b[e + 1])
        assert near(dw[e], dy[r][torch.arange(K, device="cuda") * 3 % counts[e]].T.double() * x[r].sum(0).double())


@pytest.mark.parametrize("positive", [False, True])
def test_long_sums_of_planes(positive):
    """Sums of D products: 64 of them in an accumulator that truncates (64 additions of the largest
    products and 320 of products below 2^-7 of those, a unit in the last place each), D / 64 such sums
    rounded to nearest (half a unit each), and 2^-23 for the products left out: below (68 + D / 128) *
    2^-23 of the sum of absolute products, where one accumulator would be off by up to D * 2^-23."""
    gen = torch.Generator(device="cuda").manual_seed(12)
    R, N, K = 8192, 160, 328
    off = torch.tensor([0, R], dtype=torch.int32, device="cuda")
    make = lambda *s: (lambda t: t.abs() + 0.5 if positive else t)(torch.randn(*s, generator=gen, device="cuda"))

    def check(got, a, c, depth):
        a, c = a.double(), c.double()
        assert ((got.double() - a @ c).abs() <= (68 + depth / 128) * 2.0 ** -23 * (a.abs() @ c.abs())).all()

    dy, x = make(R, N), make(R, K)
    assert _on_planes(1, R, N, K, 1)
    check(ops.grouped_gemm_wgrad(dy, x, off, 1)[0], dy.T, x, R)
    off[1] = 100
    dy, w = make(100, R), make(1, R, K)
    assert _on_planes(0, 100, R, K, 1)
    check(ops.grouped_gemm_dgrad(dy, w, off, 1), dy, w[0], R)
    dy, w = dy[:, 1:].contiguous(), w[:, 1:].transpose(1, 2).contiguous()
    assert _on_planes(2, 100, K, R - 1, 1)
    check(ops.grouped_gemm(dy, w, off, 1), dy, w[0].T, R - 1)


@pytest.mark.parametrize("K", [1032, 1027, 1536])   # rows stored whole, by words, and from 256-column tiles
def test_weight_gradient_of_planes_with_tails_beside_what_is_not_finite(K):
    """Segments of every length mod 16, whose last stage's box holds rows of the next expert, of no expert
    and of the next plane: NaN and infinities there reach the experts that hold them only."""
    counts = [i + 64 * (i % 3) for i in range(17)]
    N, head, tail = 1024, 5, 7
    dy, x, w, b, off = _inputs(counts, N, K, torch.float32, head, tail, seed=K)
    E, R = len(counts), dy.shape[0]
    assert _on_planes(1, R, N, K, E)
    want = ops.grouped_gemm_wgrad(dy, x, off, E)
    for e in range(E):
        r = slice(b[e], b[e + 1])
        _close(want[e], dy[r].double().T @ x[r].double(), dy[r].double().abs().T @ x[r].double().abs(), counts[e] + 1, e)
    dy[:head], x[:head] = float("nan"), float("inf")
    dy[b[-1]:], x[b[-1]:] = float("inf"), float("nan")
    hit = [e for e in range(E) if e % 2 == 1]
    for e in hit:
        dy[b[e]], x[b[e + 1] - 1] = float("nan"), float("-inf")   # rows at both ends of the segment
    dw = ops.grouped_gemm_wgrad(dy, x, off, E)
    for e in range(E):
        if e in hit:
            assert torch.isnan(dw[e]).all()
        else:
            assert torch.equal(dw[e], want[e])


def test_weight_gradient_of_planes_of_every_magnitude():
    """Near the largest value and tiny ones, as in test_fp32_of_every_magnitude, where the weight
    gradient runs on planes."""
    counts, N, K = [70, 33], 2048, 4104
    dy, x, w, b, off = _inputs(counts, N, K, torch.float32, seed=6)
    assert _on_planes(1, dy.shape[0], N, K, 2)
    for scale, other in ((2.0 ** 126, 2.0 ** -60), (2.0 ** -115, 2.0 ** 40), (2.0 ** -124, 2.0 ** 30), (2.0 ** 60, 2.0 ** -100)):
        d, u = dy.clamp(-3.9, 3.9) * scale, x * other
        dw = ops.grouped_gemm_wgrad(d, u, off, 2)
        for e in range(2):
            p, q = d[b[e]:b[e + 1]].double().T, u[b[e]:b[e + 1]].double()
            tol = (counts[e] + 1) * 2.0 ** -23 * (p.abs() @ q.abs()) + 2.0 ** -148
            tol = tol + 2.0 ** -134 * (q.abs().sum(0)[None] + p.abs().sum(1)[:, None])
            assert torch.isfinite(dw[e]).all() and ((dw[e].double() - p @ q).abs() <= tol).all(), (scale, other, e)


def test_weight_gradient_of_planes_at_once_replayed_and_under_a_limit():
    counts, N, K = [140, 0, 161, 5], 2048, 2056
    dy, x, w, b, off = _inputs(counts, N, K, torch.float32)
    assert _on_planes(1, dy.shape[0], N, K, 4)
    other = dy.flip(0).contiguous()
    want = [ops.grouped_gemm_wgrad(g, x, off, 4) for g in (dy, other)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(4):
        for i, g in enumerate((dy, other)):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.grouped_gemm_wgrad(g, x, off, 4))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[i]) for i in range(2) for a in got[i])
    lib = capi.lib()
    before = lib.lmoe_get_gemm_sm_limit()
    try:
        lib.lmoe_set_gemm_sm_limit(6)                # many tiles a pair
        assert torch.equal(ops.grouped_gemm_wgrad(dy, x, off, 4), want[0])
    finally:
        lib.lmoe_set_gemm_sm_limit(before)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gw = ops.grouped_gemm_wgrad(dy, x, off, 4)
    dy.copy_(other)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(gw, want[1])


@pytest.mark.parametrize("offsets", [[0, 50, 40, 100, 100], [0, 20, 40, 90, 101]])
def test_planes_and_bad_offsets(offsets):
    N, K = 2048, 2056
    dy, x, w = torch.ones(100, N, device="cuda"), torch.ones(100, K, device="cuda"), torch.ones(4, N, K, device="cuda")
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    assert _on_planes(0, 100, N, K, 4) and _on_planes(1, 100, N, K, 4)
    for call in (lambda e: ops.grouped_gemm_dgrad(dy, w, off, 4, error=e), lambda e: ops.grouped_gemm_wgrad(dy, x, off, 4, error=e)):
        e = torch.zeros(1, dtype=torch.int32, device="cuda")
        assert (call(e) == 0).all() and e.item() != 0
