"""GPU tests of the microscaled 4-bit operators against their definition in 64 bits.

Quantising and dequantising are exact (codes, scale bytes and bf16 values equal the oracle's).
The product's tolerance is derived from its arithmetic: the 4-bit products are exact, K of them
are summed in fp32 (at most K * 2^-23 of the sum of absolute products, each addition off by at
most one unit in the last place), one factor (2^-24) and one rounding to the output type
(eps / 2).  SwiGLU adds the error of the fast exponential and division.
"""
import numpy as np
import pytest
import torch

import fp4_reference as ref
from light_moe_b200 import capi, ops

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _np(t):
    return t.cpu().numpy()


def _check_quantize(x, fmt, g=None, **kw):
    q, s = ops.quantize_fp4(x, fmt, None if g is None else torch.tensor([g], device="cuda"), **kw)
    c, b = ref.quantize(x.double().cpu().numpy(), fmt, 1.0 if g is None else float(np.float32(g)))
    assert q.dtype == torch.uint8 and s.dtype == torch.uint8
    assert (_np(s) != b).sum() == 0
    assert (ref.unpack(_np(q)) != c).sum() == 0
    return q, s


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,K", [(1, 32), (3, 96), (257, 2816), (5, 4096), (2, 8224)])
def test_quantize_random(fmt, dt, rows, K):
    gen = torch.Generator(device="cuda").manual_seed(rows + K)
    x = (torch.randn(rows, K, generator=gen, device="cuda") * 3).to(DT[dt])
    x[:, ::17] *= 20
    q, s = _check_quantize(x, fmt)
    v = ops.dequantize_fp4(q, s, fmt)
    want = torch.from_numpy(ref.values(_np(q), _np(s), fmt)).to(torch.bfloat16)   # exact in both formats
    assert torch.equal(v.cpu(), want)


@pytest.mark.parametrize("g", [1.0, 0.5, 0.0123456, 3.7e-5, 1e-33, 1e35])
def test_quantize_tensor_scale(g):
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(64, 512, generator=gen, device="cuda") * (g * 100)
    q, s = _check_quantize(x, "nvfp4", g)
    v = _np(ops.dequantize_fp4(q, s, "nvfp4", torch.tensor([g], device="cuda")).double())
    want = ref.values(_np(q), _np(s), "nvfp4", float(np.float32(g)))
    # fp32 product with g, then bf16: half a unit of each (and of the smallest normal fp32)
    assert np.all(np.abs(v - want) <= (2.0 ** -8 + 2.0 ** -23) * np.abs(want) + 2.0 ** -133)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("unit", [1.0, 2.0 ** -20, 1.125, 0.3])
def test_quantize_ties_and_borders(fmt, unit):
    """Every multiple of 1/8 up to 8 and its fp32 neighbours, in units of the scale."""
    t = torch.arange(0, 65, dtype=torch.float64) / 8
    f = (t * unit).float()
    v = torch.cat([f, torch.nextafter(f, f * 0 - 1), torch.nextafter(f, f * 0 + 100)])
    v = torch.cat([v, -v])
    b = ref.BLOCK[fmt]
    per = b - 1
    n = (len(v) + per - 1) // per
    v = torch.cat([v, torch.zeros(n * per - len(v))]).view(n, per)
    top = torch.full((n, 1), 6.0 * unit)                     # nails the block's scale (MX: at most 8 -> 2 units)
    x = torch.cat([top, v.clamp(-6.0 * unit, 6.0 * unit)], 1).view(1, -1)
    x = torch.cat([x, torch.zeros(1, (-x.shape[1]) % 32)], 1)
    x = x.cuda()
    _check_quantize(x, fmt)
    if fmt == "nvfp4":
        for g in (0.75, 1 / 3, 0.01):
            _check_quantize((x * g).contiguous(), fmt, g)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_quantize_extremes(fmt):
    x = torch.zeros(8, 64, device="cuda")
    x[0, 3] = 3.0e38
    x[1] = 1e-45
    x[2] = -1.17549435e-38
    x[3, ::2] = 5e-39
    x[4] = -0.0
    x[5, 0], x[5, 1] = 448.0 * 6, 500.0 * 6
    x[6] = 2.0 ** -9 * 6
    x[7] = 2.0 ** -10 * 6
    _check_quantize(x, fmt)
    _check_quantize(x.to(torch.bfloat16), fmt)


@pytest.mark.parametrize("fmt,nan_byte", [("mxfp4", 255), ("nvfp4", 127)])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_quantize_blocks_that_are_not_finite(fmt, nan_byte, dt, bad):
    x = torch.ones(3, 128, device="cuda", dtype=DT[dt])
    x[1, 70] = bad
    q, s = _check_quantize(x, fmt)
    blk = 70 // ref.BLOCK[fmt]
    assert s[1, blk].item() == nan_byte and (s == nan_byte).sum().item() == 1
    v = ops.dequantize_fp4(q, s, fmt)
    assert torch.isnan(v).sum().item() == ref.BLOCK[fmt]


@pytest.mark.parametrize("g", [0.0, -1.0, float("nan"), float("inf")])
def test_quantize_bad_tensor_scale_gives_nan(g):
    x = torch.ones(2, 32, device="cuda")
    q, s = ops.quantize_fp4(x, "nvfp4", torch.tensor([g], device="cuda"))
    assert (s == 127).all() and (q == 0).all()


def test_quantize_views_batches_and_scales_per_expert():
    gen = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.randn(40, 400, generator=gen, device="cuda").to(torch.bfloat16)
    for v in (wide[:, 8:8 + 96], wide[:, 3:3 + 96], wide[::3, :64], wide[:, ::2][:, :96], wide.t()[:64, :32]):
        _check_quantize(v, "mxfp4")
        _check_quantize(v, "nvfp4")
    w = torch.randn(3, 5, 64, generator=gen, device="cuda")
    g = torch.tensor([0.5, 0.01, 2.0], device="cuda")
    q, s = ops.quantize_fp4(w, "nvfp4", g)
    assert q.shape == (3, 5, 32) and s.shape == (3, 5, 4)
    v = ops.dequantize_fp4(q, s, "nvfp4", g)
    for e in range(3):
        c, b = ref.quantize(w[e].double().cpu().numpy(), "nvfp4", float(g[e]))
        assert np.array_equal(ref.unpack(_np(q[e])), c) and np.array_equal(_np(s[e]), b)
        assert torch.equal(v[e], ops.dequantize_fp4(q[e], s[e], "nvfp4", g[e:e + 1]))
    q0, s0 = ops.quantize_fp4(torch.empty(0, 64, device="cuda"), "mxfp4")
    assert q0.shape == (0, 32) and ops.dequantize_fp4(q0, s0, "mxfp4").shape == (0, 64)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_quantize_to_permuted_rows(fmt):
    """Row r lands on every row of positions[r]; entries outside the output are skipped."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    T, k, K = 37, 3, 160
    x = torch.randn(T, K, generator=gen, device="cuda").to(torch.bfloat16)
    pos = torch.randperm(T * k, generator=torch.Generator().manual_seed(3)).to(torch.int32).view(T, k).cuda()
    q1, s1 = ops.quantize_fp4(x, fmt)
    q, s = ops.quantize_fp4(x, fmt, positions=pos)
    assert q.shape == (T * k, K // 2)
    for j in range(k):
        assert torch.equal(q[pos[:, j].long()], q1) and torch.equal(s[pos[:, j].long()], s1)
    # the caller's buffers behind the last row stay as they are
    pitch = capi.lib().lmoe_fp4_scale_pitch(K, capi.LMOE_FP4_MX if fmt == "mxfp4" else capi.LMOE_FP4_NV)
    qb = torch.full((T * k + 2, K // 2), 7, dtype=torch.uint8, device="cuda")
    sb = torch.full((T * k + 2, pitch), 7, dtype=torch.uint8, device="cuda")
    bad = pos.clone()
    bad[0, 0], bad[1, 1] = -1, T * k
    capi.call("lmoe_quantize_fp4", x.data_ptr(), 0, T, K, K, 0 if fmt == "mxfp4" else 1, None, 1, bad.data_ptr(), k,
              T * k, qb.data_ptr(), sb.data_ptr(), capi.stream_handle())
    assert (qb[T * k:] == 7).all() and (sb[T * k:] == 7).all()
    hit = torch.ones(T * k, dtype=torch.bool)
    hit[pos[0, 0].item()] = hit[pos[1, 1].item()] = False
    assert torch.equal(qb[:T * k].cpu()[hit], q.cpu()[hit]) and (qb[:T * k].cpu()[~hit] == 7).all()
    assert (sb[:T * k].cpu()[hit][:, K // ref.BLOCK[fmt]:] == 0).all()   # the padding of a scale row


def test_refusals_on_the_device():
    x = torch.ones(4, 64, device="cuda")
    q, s = ops.quantize_fp4(x, "mxfp4")
    off = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    g1 = torch.ones(1, device="cuda")
    for call in (
        lambda: ops.quantize_fp4(x, "fp4"),
        lambda: ops.quantize_fp4(x[:, :40], "mxfp4"),
        lambda: ops.quantize_fp4(x.double(), "mxfp4"),
        lambda: ops.quantize_fp4(x[0], "mxfp4"),
        lambda: ops.quantize_fp4(x, "mxfp4", g1),
        lambda: ops.quantize_fp4(x, "nvfp4", g1.double()),
        lambda: ops.quantize_fp4(x, "nvfp4", torch.ones(4, device="cuda")),
        lambda: ops.quantize_fp4(x, "nvfp4", torch.ones(1)),
        lambda: ops.quantize_fp4(x, "mxfp4", positions=torch.arange(4, device="cuda")),
        lambda: ops.quantize_fp4(x, "mxfp4", positions=torch.arange(5, dtype=torch.int32, device="cuda")),
        lambda: ops.dequantize_fp4(q, s[:, :1], "mxfp4"),
        lambda: ops.dequantize_fp4(q, s[:3], "mxfp4"),
        lambda: ops.dequantize_fp4(q.int(), s, "mxfp4"),
        lambda: ops.fp4_grouped_gemm(q, s, q[None, :, :16], s[None], off, 1, "mxfp4"),
        lambda: ops.fp4_grouped_gemm(q, s, q[None], s[None], off, 2, "mxfp4"),
        lambda: ops.fp4_grouped_gemm(q, s, q[None], s[None], off, 0, "mxfp4"),
        lambda: ops.fp4_grouped_gemm(q, s, q[None], s[None], off.float(), 1, "mxfp4"),
        lambda: ops.fp4_grouped_gemm(q, s, q[None], s[None], off.cpu(), 1, "mxfp4"),
        lambda: ops.fp4_grouped_gemm(q, s, q[None], s[None], off, 1, "nvfp4"),
        lambda: ops.fp4_grouped_gemm(q, s, q[None], s[None], off, 1, "mxfp4", weights_up=q[None]),
        lambda: ops.fp4_grouped_gemm(q, s, q[None], s[None], off, 1, "mxfp4", alpha_up=g1),
        lambda: ops.fp4_grouped_gemm(q, s, q[None], s[None], off, 1, "mxfp4", alpha=g1.double()),
        lambda: ops.fp4_grouped_gemm(q, s, q[None], s[None], off, 1, "mxfp4", out_dtype=torch.float64),
    ):
        with pytest.raises(RuntimeError):
            call()


# ------------------------------------------------------------------------------------ product
def _operand(shape, fmt, gen, std=1.0):
    x = torch.randn(*shape, generator=gen, device="cuda") * std
    return ops.quantize_fp4(x, fmt)


def _product64(xq, xs, wq, ws, bounds, fmt, alpha=None):
    """Sums and sums of absolute products, in 64 bits, zero outside the experts."""
    x = torch.from_numpy(ref.values(_np(xq), _np(xs), fmt)).cuda()
    w = torch.from_numpy(ref.values(_np(wq), _np(ws), fmt)).cuda()
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device="cuda")
    m = torch.zeros_like(y)
    for e in range(len(bounds) - 1):
        a, b = bounds[e], bounds[e + 1]
        f = 1.0 if alpha is None else float(alpha[e])
        y[a:b] = x[a:b] @ w[e].T * f
        m[a:b] = x[a:b].abs() @ w[e].abs().T * abs(f)
    return y, m


def _check_product(counts, N, K, fmt, swiglu=False, odt=torch.bfloat16, head=0, tail=0, i64=False, alpha=True, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    E = len(counts)
    bounds = [head]
    for c in counts:
        bounds.append(bounds[-1] + c)
    R = bounds[-1] + tail
    off = torch.tensor(bounds, dtype=torch.int64 if i64 else torch.int32, device="cuda")
    xq, xs = _operand((R, K), fmt, gen)
    wq, ws = _operand((E, N, K), fmt, gen, 0.1)
    al = (torch.rand(E, generator=gen, device="cuda") + 0.5) if alpha else None
    kw = {}
    if swiglu:
        uq, us = _operand((E, N, K), fmt, gen, 0.1)
        au = (torch.rand(E, generator=gen, device="cuda") + 0.5) if alpha else None
        kw = dict(weights_up=uq, weight_scales_up=us, alpha_up=au)
    y = ops.fp4_grouped_gemm(xq, xs, wq, ws, off, E, fmt, alpha=al, out_dtype=odt, **kw)
    assert y.dtype == odt and y.shape == (R, N)
    half = torch.finfo(odt).eps / 2
    acc = (K + 2) * 2.0 ** -23
    g, mg = _product64(xq, xs, wq, ws, bounds, fmt, al)
    if swiglu:
        u, mu = _product64(xq, xs, uq, us, bounds, fmt, au)
        dg, du = acc * mg, acc * mu
        want = g * torch.sigmoid(g) * u
        # |silu'| <= 1.1; exp off by 2 + 1.16 |g| units, the division by 2
        fast = (6 + 1.16 * g.abs()) * 2.0 ** -23
        off_by = 1.1 * dg * (u.abs() + du) + (g.abs() + dg) * du + fast * want.abs()
    else:
        want, off_by = g, acc * mg
    tol = off_by * (1 + half) + half * want.abs() + torch.finfo(odt).tiny
    bad = (y.double() - want).abs() > tol
    assert not bad.any(), (bad.sum().item(), (y.double() - want).abs().max().item())
    assert (y[:head] == 0).all() and (y[R - tail:] == 0).all()


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("counts,N,K", [
    ([1], 64, 64), ([1, 0, 3], 96, 128), ([128], 192, 256), ([256, 129, 0, 31], 200, 512), ([5, 300], 384, 1408),
    ([17, 33, 65], 1000, 96), ([2, 2], 7, 32), ([700], 640, 2816),
])
def test_product(fmt, swiglu, counts, N, K):
    _check_product(counts, N, K, fmt, swiglu)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("odt", [torch.bfloat16, torch.float16, torch.float32])
def test_product_output_types(fmt, odt):
    _check_product([40, 200], 300, 320, fmt, odt=odt)
    _check_product([40, 200], 160, 320, fmt, swiglu=True, odt=odt, alpha=False)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("swiglu", [False, True])
def test_product_rows_outside_experts_and_offsets_64(fmt, swiglu):
    _check_product([60, 0, 300, 1], 250, 608, fmt, swiglu, head=3, tail=290, i64=True)
    _check_product([0, 0], 192, 256, fmt, swiglu, head=0, tail=5)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_product_many_experts_and_long_sums(fmt):
    _check_product([i % 7 for i in range(256)], 64, 64, fmt)
    _check_product([9, 140], 256, 14336, fmt)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_nan_blocks_stay_in_their_rows(fmt):
    """A NaN block reaches its own row (or its weight's column) only; rows of other experts that
    share a tile, padding bytes of scale rows and rows outside the experts do not leak."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    R, N, K = 200, 130, 160
    x = torch.randn(R, K, generator=gen, device="cuda")
    w = torch.randn(2, N, K, generator=gen, device="cuda")
    off = torch.tensor([10, 90, 180], dtype=torch.int32, device="cuda")
    clean = ops.fp4_grouped_gemm(*ops.quantize_fp4(x, fmt), *ops.quantize_fp4(w, fmt), off, 2, fmt)
    x[5], x[50, 33], x[185, 0] = float("nan"), float("inf"), float("nan")
    w[1, 7, 100] = float("nan")
    xq, xs = ops.quantize_fp4(x, fmt)
    wq, ws = ops.quantize_fp4(w, fmt)
    # padding bytes of both scale rows hold the NaN byte
    fill = 255 if fmt == "mxfp4" else 127
    xs.as_strided((R, 32), (xs.stride(0), 1))[:, K // ref.BLOCK[fmt]:] = fill
    ws.as_strided((2, N, 32), (ws.stride(0), ws.stride(1), 1))[..., K // ref.BLOCK[fmt]:] = fill
    y = ops.fp4_grouped_gemm(xq, xs, wq, ws, off, 2, fmt)
    want = torch.zeros(R, N, dtype=torch.bool, device="cuda")
    want[50] = True
    want[90:180, 7] = True
    assert torch.equal(torch.isnan(y), want)
    assert torch.equal(y[~want], clean[~want])
    assert (y[:10] == 0).all() and (y[180:] == 0).all()


@pytest.mark.parametrize("offsets", [[0, 50, 40, 100], [-1, 20, 40, 100], [0, 20, 40, 101]])
def test_bad_offsets_give_zeros_and_an_error_word(offsets):
    R, N, K = 100, 64, 64
    xq, xs = ops.quantize_fp4(torch.ones(R, K, device="cuda"), "mxfp4")
    wq, ws = ops.quantize_fp4(torch.ones(3, N, K, device="cuda"), "mxfp4")
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    y = torch.full((R, N), 5.0, device="cuda", dtype=torch.bfloat16)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    capi.call("lmoe_fp4_grouped_gemm", xq.data_ptr(), xs.data_ptr(), 32, R, K, wq.data_ptr(), ws.data_ptr(), None,
              None, 32, N, 0, off.data_ptr(), 0, 3, None, None, 0, y.data_ptr(), err.data_ptr(), capi.stream_handle())
    assert (y == 0).all() and err.item() != 0


def test_scales_on_other_pitches_and_views_of_codes():
    gen = torch.Generator(device="cuda").manual_seed(4)
    R, N, K, fmt = 70, 96, 320, "nvfp4"
    off = torch.tensor([0, 30, 70], dtype=torch.int32, device="cuda")
    xq, xs = _operand((R, K), fmt, gen)
    wq, ws = _operand((2, N, K), fmt, gen)
    uq, us = _operand((2, N, K), fmt, gen)
    want = ops.fp4_grouped_gemm(xq, xs, wq, ws, off, 2, fmt)
    both = ops.fp4_grouped_gemm(xq, xs, wq, ws, off, 2, fmt, weights_up=uq, weight_scales_up=us)
    xsc, wsc = xs.contiguous(), ws.contiguous()                      # 20 bytes a row
    assert torch.equal(ops.fp4_grouped_gemm(xq, xsc, wq, wsc, off, 2, fmt), want)
    wide = torch.zeros(2, N, 64, dtype=torch.uint8, device="cuda")   # another pitch of 32s
    wide[..., :20] = ws
    assert torch.equal(ops.fp4_grouped_gemm(xq, xs, wq, wide[..., :20], off, 2, fmt), want)
    assert torch.equal(ops.fp4_grouped_gemm(xq, xs, wq, wide[..., :20], off, 2, fmt, weights_up=uq,
                                            weight_scales_up=us), both)
    assert torch.equal(ops.fp4_grouped_gemm(xq, xs, wq, ws, off, 2, fmt, weights_up=uq,
                                            weight_scales_up=us.contiguous()), both)
    xw = torch.zeros(R, K // 2 + 3, dtype=torch.uint8, device="cuda")
    xw[:, 3:] = xq
    assert torch.equal(ops.fp4_grouped_gemm(xw[:, 3:], xs, wq, ws, off, 2, fmt), want)
    exact = torch.zeros(R * 32 - 12, dtype=torch.uint8, device="cuda")   # storage ends with the last row's scales
    last = exact.as_strided((R, 20), (32, 1))
    last.copy_(xs)
    assert torch.equal(ops.fp4_grouped_gemm(xq, last, wq, ws, off, 2, fmt), want)
    more = ops.fp4_grouped_gemm(xq, xs, wq, ws, off[:2], 1, fmt)     # fewer experts than weights
    assert torch.equal(more[:30], want[:30]) and (more[30:] == 0).all()


def test_streams_graphs_and_the_sm_limit():
    gen = torch.Generator(device="cuda").manual_seed(6)
    R, N, K, fmt = 300, 500, 640, "mxfp4"
    off = torch.tensor([0, 130, 300], dtype=torch.int32, device="cuda")
    x = torch.randn(R, K, generator=gen, device="cuda").to(torch.bfloat16)
    wq, ws = _operand((2, N, K), fmt, gen)

    def step():
        xq, xs = ops.quantize_fp4(x, fmt)
        return ops.fp4_grouped_gemm(xq, xs, wq, ws, off, 2, fmt)

    want = step()
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s1):
        a = step()
    with torch.cuda.stream(s2):
        b = step()
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    x.copy_(x.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, step())
    lib = capi.lib()
    before = lib.lmoe_get_gemm_sm_limit()
    try:
        for cap in (1, 3, 64):
            lib.lmoe_set_gemm_sm_limit(cap)
            assert torch.equal(step(), y)
    finally:
        lib.lmoe_set_gemm_sm_limit(before)


@pytest.mark.parametrize("odt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("N", [8, 40, 104, 264])
def test_blocks_of_rows_cut_by_the_last_column(odt, swiglu, N):
    """Whole blocks of 32 rows leave together, also where the output ends inside a block."""
    _check_product([200, 0, 96, 165], N, 96, "mxfp4", swiglu, odt=odt, head=7, tail=40, seed=N)


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("shift", [2, 16, 32])
def test_output_anywhere_and_nothing_beside_it(swiglu, shift):
    """An output at an address of `shift` bytes behind a 256-byte boundary; bytes around it stay."""
    gen = torch.Generator(device="cuda").manual_seed(shift)
    R, N, K, fmt = 300, 136, 128, "nvfp4"
    off = torch.tensor([0, 130, 300], dtype=torch.int32, device="cuda")
    xq, xs = _operand((R, K), fmt, gen)
    wq, ws = _operand((2, N, K), fmt, gen)
    up = dict(weights_up=wq, weight_scales_up=ws) if swiglu else {}
    want = ops.fp4_grouped_gemm(xq, xs, wq, ws, off, 2, fmt, **up)
    buf = torch.full((R * N * 2 + 512,), 0x5A, dtype=torch.uint8, device="cuda")
    u = (wq.data_ptr(), ws.data_ptr()) if swiglu else (None, None)
    capi.call("lmoe_fp4_grouped_gemm", xq.data_ptr(), xs.data_ptr(), 32, R, K, wq.data_ptr(), ws.data_ptr(), *u, 32, N, 1,
              off.data_ptr(), 0, 2, None, None, 0, buf.data_ptr() + 256 + shift, None, capi.stream_handle())
    y = buf[256 + shift:256 + shift + R * N * 2]
    assert torch.equal(y, want.view(torch.uint8).flatten())
    assert (buf[:256 + shift] == 0x5A).all() and (buf[256 + shift + R * N * 2:] == 0x5A).all()


def test_scales_at_odd_addresses():
    gen = torch.Generator(device="cuda").manual_seed(6)
    R, N, K, fmt = 90, 64, 512, "nvfp4"
    off = torch.tensor([0, 90], dtype=torch.int32, device="cuda")
    xq, xs = _operand((R, K), fmt, gen)
    wq, ws = _operand((1, N, K), fmt, gen)
    want = ops.fp4_grouped_gemm(xq, xs, wq, ws, off, 1, fmt)
    for shift in (1, 16):
        moved = torch.zeros(R * 32 + shift, dtype=torch.uint8, device="cuda")[shift:].view(R, 32)
        moved.copy_(xs)
        assert torch.equal(ops.fp4_grouped_gemm(xq, moved, wq, ws, off, 1, fmt), want)


def test_broadcast_scales():
    """Scales that are one row for many (stride 0), in either leading dimension."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    E, N, K, fmt = 3, 40, 64, "mxfp4"
    q = torch.randint(0, 256, (E, N, K // 2), generator=gen, device="cuda", dtype=torch.uint8)
    xq, xs = _operand((70, K), fmt, gen)
    off = torch.tensor([0, 20, 25, 70], dtype=torch.int32, device="cuda")
    for shape in ((E, 1, 32), (1, N, 32), (1, 1, 32)):
        rows = torch.randint(120, 130, shape, generator=gen, device="cuda", dtype=torch.uint8)
        s = rows[..., :K // 32].expand(E, N, K // 32)
        assert torch.equal(ops.dequantize_fp4(q, s, fmt), ops.dequantize_fp4(q, s.contiguous(), fmt))
        assert torch.equal(ops.fp4_grouped_gemm(xq, xs, q, s, off, E, fmt),
                           ops.fp4_grouped_gemm(xq, xs, q, s.contiguous(), off, E, fmt))


def test_quantize_borders_of_tiny_and_short_values():
    """Values at the borders between codes: fp32 ones so small that their distance from a border lies
    below the smallest fp32, and 16-bit ones that meet borders exactly, under scales of every mantissa."""
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    gen = np.random.default_rng(3)
    rows = []
    g = np.float32(1.37e-37)
    for c in np.concatenate([np.arange(8, 16) / 8, np.arange(8, 16) * 4]):
        d = np.float64(g) * c
        v = (borders * d).astype(np.float32)
        near = np.concatenate([v, np.nextafter(v, np.float32(1))])
        rows.append(np.concatenate([[np.float32(6 * d)], near, [0]]) * gen.choice([-1, 1], 16))
    x = torch.from_numpy(np.array(rows, dtype=np.float32)).reshape(-1, 32).cuda()
    _check_quantize(x, "nvfp4", float(g))
    for dt in (torch.bfloat16, torch.float16):
        for g in (None, 1.0, 0.25, 8.0, 0.3):
            rows = []
            for c in np.arange(8, 16) / 8 * (1.0 if g is None else g):
                for k in range(8):
                    v = borders * c * 2.0 ** gen.integers(-1, 2, 7)
                    rows.append(np.concatenate([[6 * c], v, [6 * c * (k + 8.5) / 16], gen.standard_normal(7) * c]))
            x = torch.from_numpy(np.array(rows)).to(dt).reshape(-1, 32).cuda()
            _check_quantize(x, "nvfp4", g)


def test_quantize_scales_at_midpoints():
    """Largest values whose sixth lies half way between two scales, in every type."""
    for dt in DT.values():
        for g in (None, 0.5, 0.7):
            n = np.arange(0, 16) + 0.5
            top = np.concatenate([6 * n * 2.0 ** e for e in (-9, -6, -3, 0, 3)]) * (1.0 if g is None else g)
            x = torch.zeros(80, 16, dtype=torch.float64)
            x[:, 3] = torch.from_numpy(top)
            x[:, 5] = x[:, 3] / 3
            _check_quantize(x.to(dt).reshape(-1, 32).cuda(), "nvfp4", g)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_quantize_keeps_the_sign_of_zeros_and_tiny_values(fmt, dt):
    x = torch.zeros(4, 64)
    x[:, ::8] = 6.0
    x[:, 1::4] = -0.0
    x[:, 2::4] = -6e-8
    x[2:, 3::4] = -1.0
    x[3] = -0.0
    _check_quantize(x.to(DT[dt]).cuda(), fmt)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("g", [2.0 ** e for e in (-126, -120, -100, -80, -64, -30, -20, -12, -10, -9, -8, -4, 0, 20, 100)]
                         + [0.3, 3.7e-5, 1e-33])
def test_quantize_saturates_values_far_beyond_the_range(dt, g):
    """Values of both signs up to the largest of their type, alone and beside values at the borders
    between codes, under a scale at its limit of 448."""
    gen = np.random.default_rng(5)
    big = float(torch.finfo(torch.bfloat16).max)
    rows = []
    for top in (big, big / 2, 2.0 ** 100, 1.0, 448 * 6 * g, 448 * 6 * g * 1.0625, 448 * 8 * g, 448 * 8 * g * 1.125,
                448 * g * 2.0 ** 20):
        for lone in (top, -top):
            v = gen.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 1.0, -2.5, -5.0, -0.0], 16) * 448 * g
            v[3] = lone
            rows += [v, np.full(16, lone)]
    x = torch.from_numpy(np.clip(np.array(rows), -big, big)).to(torch.bfloat16).to(DT[dt]).reshape(-1, 32).cuda()
    _check_quantize(x, "nvfp4", g)
    if dt == "fp32":
        _check_quantize(torch.nextafter(x, x * 0), "nvfp4", g)   # every bit of the mantissa in use


@pytest.mark.parametrize("shape", [(0, 4, 64), (3, 0, 64), (0, 64)])
def test_empty_batches_with_their_tensor_scales(shape):
    """No matrices and no scales, no rows under a scale each, and one scale for nothing."""
    lead = shape[0] if len(shape) == 3 else 1
    for n in {lead, 1}:
        g = torch.ones(n, device="cuda")
        q, s = ops.quantize_fp4(torch.empty(shape, device="cuda"), "nvfp4", g)
        assert q.shape == shape[:-1] + (32,) and s.shape == shape[:-1] + (4,)
        assert ops.dequantize_fp4(q, s, "nvfp4", g).shape == shape


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_quantize_the_longest_row(fmt):
    """K = 2^31 - 32: the padded scale row stands for 2^31 values."""
    K = 2 ** 31 - 32
    x = torch.zeros(1, K, device="cuda", dtype=torch.bfloat16)
    places = torch.tensor([0, 40, 2 ** 30 + 64, K - 1], device="cuda")
    x[0, places] = torch.tensor([6.0, -3.0, 1.5, 4.0], device="cuda", dtype=torch.bfloat16)
    q, s = ops.quantize_fp4(x, fmt)
    assert q.shape == (1, K // 2) and s.shape == (1, K // ref.BLOCK[fmt])
    v = ops.dequantize_fp4(q, s, fmt)
    if fmt == "nvfp4":
        x[0, K - 1] = 4.125   # 4 / 6 has the scale 0.6875, between 0.625 and 0.6875, and 4 / 0.6875 the code 6
    assert torch.equal(v, x)


@pytest.mark.parametrize("rows", [100, 400])   # one for each kernel
def test_error_words_of_the_product(rows):
    x, w = ops.quantize_fp4(torch.ones(rows, 64, device="cuda"), "mxfp4"), ops.quantize_fp4(torch.ones(3, 40, 64, device="cuda"), "mxfp4")
    for offsets, bad in (([0, 50, 40, rows], True), ([0, 20, 40, rows + 1], True), ([0, 20, 40, rows], False)):
        off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
        e = torch.zeros(1, dtype=torch.int32, device="cuda")
        y = ops.fp4_grouped_gemm(*x, *w, off, 3, "mxfp4", error=e)
        assert (e.item() != 0) == bad and (y != 0).any().item() != bad
    with pytest.raises(RuntimeError):
        ops.fp4_grouped_gemm(*x, *w, off, 3, "mxfp4", error=e.float())


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("limit", [2, 0])
def test_swiglu_of_many_tiles_a_pair(fmt, limit):
    """Several tiles on each pair of CTAs, so that accumulators, exchange buffers and scales are handed
    back and used again: all tiles on one pair, and more than three rounds on all of them."""
    lib = capi.lib()
    before = lib.lmoe_get_gemm_sm_limit()
    try:
        lib.lmoe_set_gemm_sm_limit(limit)
        few = [i % 3 for i in range(64)]             # the kernel for few rows; one expert with two tiles of rows
        few[5], few[40] = 70, 0
        _check_product(few, 200 if limit else 1000, 160, fmt, swiglu=True, head=3, tail=5)
        _check_product(few, 200 if limit else 1000, 1056, fmt, swiglu=True, odt=torch.float32)
        many = [700, 0, 300, 129]
        _check_product(many, 1000 if limit else 4096, 96, fmt, swiglu=True, head=300, tail=40)
        _check_product(many, 1000 if limit else 4096, 608, fmt, swiglu=True, odt=torch.float32)
    finally:
        lib.lmoe_set_gemm_sm_limit(before)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("odt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("N,K", [(200, 32), (7, 96), (384, 1408), (264, 14336)])
def test_both_kernels_give_the_same_bits(fmt, odt, swiglu, N, K):
    """The rule chooses by all rows, so rows outside the experts move a call to the other kernel: what a
    row gives does not depend on how many come with it."""
    gen = torch.Generator(device="cuda").manual_seed(N + K)
    counts = [1, 0, 70, 3, 33]
    E, R = len(counts), sum(counts)
    few = E * (32 if swiglu else 64)
    off = torch.tensor(np.cumsum([0] + counts), dtype=torch.int32, device="cuda")
    xq, xs = _operand((few + 64, K), fmt, gen)
    wq, ws = _operand((E, N, K), fmt, gen, 0.1)
    al = torch.rand(E, generator=gen, device="cuda") + 0.5
    kw = dict(alpha=al, out_dtype=odt)
    if swiglu:
        uq, us = _operand((E, N, K), fmt, gen, 0.1)
        kw.update(weights_up=uq, weight_scales_up=us, alpha_up=al * 0.7)
    a = ops.fp4_grouped_gemm(xq[:R], xs[:R], wq, ws, off, E, fmt, **kw)
    b = ops.fp4_grouped_gemm(xq, xs, wq, ws, off, E, fmt, **kw)
    assert torch.equal(a, b[:R]) and (b[R:] == 0).all()
