"""GPU tests of the 8-bit floating-point operators against their definition in 64 bits.

Quantising is exact (codes and scales equal the reference's); dequantising rounds a product to fp32
and then to the output type.  The product's tolerance is derived from its arithmetic: the products of
codes are exact; 128 of them are summed in fp32 (at most 2^-23 of the sum of absolute values for
each addition, which may truncate); the two scales' product, its product with that sum and the sum
over the blocks round to nearest (2^-24 each); one rounding to the output type (eps / 2).  SwiGLU
adds the error of the fast exponential and division.
"""
import numpy as np
import pytest
import torch

import fp8_reference as ref
from light_moe_b200 import capi, ops

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}


def _np(t):
    return t.double().cpu().numpy()


def _check(x, block_rows=1, power_of_two=False):
    """quantize_fp8 of a 2-D tensor equals the definition."""
    q, s = ops.quantize_fp8(x, block_rows=block_rows, power_of_two=power_of_two)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape
    assert s.dtype == torch.float32 and s.shape == (-(-x.shape[0] // block_rows), ref.blocks(x.shape[1]))
    want_q, want_s = ref.quantize(_np(x), block_rows, power_of_two)
    assert np.array_equal(_np(s), want_s.astype(np.float64), equal_nan=True)
    assert np.array_equal(_np(q), want_q)
    return q, s


# --------------------------------------------------------------------------------- quantise
@pytest.mark.parametrize("power", [False, True])
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("block_rows,rows,K", [(1, 1, 16), (1, 3, 144), (1, 257, 2816), (1, 5, 4096), (1, 2, 8208),
                                               (128, 1, 16), (128, 127, 128), (128, 130, 208), (128, 300, 1408)])
def test_quantize_random(block_rows, rows, K, dt, power):
    gen = torch.Generator(device="cuda").manual_seed(rows + K)
    x = (torch.randn(rows, K, generator=gen, device="cuda") * 3).to(DT[dt])
    x[:, ::17] *= 20
    q, s = _check(x, block_rows, power)
    want = ref.values(_np(q), _np(s), block_rows)
    for out in DT:
        v = ops.dequantize_fp8(q, s, block_rows=block_rows, out_dtype=DT[out])
        assert v.dtype == DT[out] and v.shape == x.shape
        # the product to fp32 (2^-24), then the type (fp32: no second rounding); 2^-25 for fp16's subnormals
        assert np.all(np.abs(_np(v) - want) <= (HALF[out] * 1.001 + 2.0 ** -24) * np.abs(want)
                      + (2.0 ** -25 if out == "fp16" else 2.0 ** -140))
    assert ops.dequantize_fp8(q, s, block_rows=block_rows).dtype == torch.bfloat16


@pytest.mark.parametrize("unit", [1.0, 2.0 ** -20, 1.125, 0.3, 1e30, 3e-38])
def test_quantize_ties_and_borders(unit):
    """Every midpoint of two codes and its fp32 neighbours, in units of the scale."""
    mid = torch.from_numpy((ref.GRID[1:] + ref.GRID[:-1]) / 2)
    grid = torch.from_numpy(ref.GRID)
    s = ref.scale(np.array([448.0 * np.float32(unit)]))[0]
    t = (torch.cat([mid, grid]) * float(s)).float()
    v = torch.cat([t, torch.nextafter(t, t * 0 - 1), torch.nextafter(t, t * 0 + 3e38)])
    v = torch.cat([v, -v])
    top = float(np.float32(448.0 * np.float32(unit)))
    v = v.clamp(-top, top)
    n = -(-len(v) // 127)
    v = torch.cat([v, torch.zeros(n * 127 - len(v))]).view(n, 127)
    x = torch.cat([torch.full((n, 1), top), v], 1).cuda()
    _check(x)
    _check(x.view(1, -1))
    _check(x, 128)
    _check(x, 1, True)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("top", [63 * 2.0 ** 122, 1.8e38, 3.0e38, 3.4028234663852886e38])
def test_quantize_ties_and_borders_at_the_end_of_fp32(top, block_rows):
    """Midpoints, codes and their fp32 neighbours in blocks whose values' doubles are infinite."""
    s = float(ref.scale(np.array([top]))[0])
    t = torch.from_numpy(np.concatenate([(ref.GRID[1:] + ref.GRID[:-1]) / 2, ref.GRID]) * s).clamp(max=top).float()
    v = [t]
    for way in (0.0, 3.4028234663852886e38):
        u = t
        for _ in range(2):
            u = torch.nextafter(u, torch.full_like(t, way))
            v.append(u)
    v = torch.cat(v).clamp(max=top)
    v = torch.cat([v, -v])
    n = -(-len(v) // 127)
    v = torch.cat([v, torch.zeros(n * 127 - len(v))]).view(n, 127)
    x = torch.cat([torch.full((n, 1), top), v], 1).cuda()
    assert (x.abs() >= 2.0 ** 127).any() and torch.isfinite(x).all()
    _check(x, block_rows)
    _check(x, block_rows, True)


@pytest.mark.parametrize("seed", range(4))
def test_quantize_many_bit_patterns(seed):
    """fp32 values of every magnitude, and 16-bit values in blocks of every top: quotients near borders."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    bits = torch.randint(0, 2 ** 32, (64, 1024), generator=gen, device="cuda").sub(2 ** 31).to(torch.int32)
    x = bits.view(torch.float32)
    x = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    _check(x)
    m = torch.randint(0, 2 ** 15, (64, 1024), generator=gen, device="cuda").to(torch.int16)
    for t in (torch.bfloat16, torch.float16):
        y = m.view(t)
        _check(torch.where(torch.isfinite(y), y, torch.zeros_like(y)))
    near = 1.0 + torch.rand(256, 512, generator=gen, device="cuda")
    _check(near.to(torch.bfloat16))
    _check(near)


@pytest.mark.parametrize("dt,bits,up", [("bf16", 8, 1.0), ("bf16", 8, 2.0 ** 100), ("bf16", 8, 2.0 ** -110), ("fp16", 11, 16.0)])
def test_quantize_16_bit_neighbours_of_every_midpoint(dt, bits, up):
    """Blocks of every significand of the largest value, and around each midpoint times the scale the type's values."""
    tops = np.arange(2 ** (bits - 1), 2 ** bits) * up
    mid = (ref.GRID[1:] + ref.GRID[:-1]) / 2
    near = torch.from_numpy(np.outer(tops / 448, mid)).float().to(DT[dt])
    top = torch.from_numpy(tops).float().to(DT[dt])[:, None]
    for step in (-1, 0, 1):   # (positive: the next patterns are the next values)
        v = (near.view(torch.int16) + step).view(DT[dt]).clamp(min=0)
        x = torch.cat([top, torch.minimum(v, top), -top], 1).cuda()
        assert x.shape[1] == 128
        _check(x)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_extremes(block_rows):
    x = torch.zeros(8, 256, device="cuda")
    x[0, 3] = 3.0e38
    x[1, :128] = 1e-45
    x[2] = -1.17549435e-38
    x[3, ::2] = 5e-39
    x[4] = -0.0
    x[5, 0], x[5, 1] = 448.0, 449.0
    for i in range(8) if block_rows > 1 else (slice(None),):
        part = x[i:i + 1] if block_rows > 1 else x
        _check(part.contiguous(), block_rows)
        _check(part.contiguous(), block_rows, True)
    _check(x.to(torch.bfloat16), block_rows)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_quantize_blocks_that_are_not_finite(block_rows, dt, bad):
    x = torch.ones(3, 300 // 16 * 16, device="cuda", dtype=DT[dt])
    x[1, 200] = bad
    q, s = _check(x, block_rows)
    assert torch.isnan(s).sum().item() == 1 and torch.isnan(s[1 // block_rows, 1])
    v = ops.dequantize_fp8(q, s, block_rows=block_rows)
    assert torch.isnan(v).sum().item() == (128 if block_rows == 1 else 3 * 128)


def test_quantize_views_batches_and_strides():
    gen = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.randn(140, 400, generator=gen, device="cuda").to(torch.bfloat16)
    for v in (wide[:, 8:8 + 96], wide[:, 3:3 + 96], wide[::3, :64], wide[:, ::2][:, :96], wide.t()[:64, :32]):
        _check(v)
        _check(v, 128)
    w = torch.randn(3, 5, 144, generator=gen, device="cuda")
    q, s = ops.quantize_fp8(w)
    assert s.shape == (3, 5, 2)
    for i in range(3):
        want_q, want_s = ref.quantize(_np(w[i]))
        assert np.array_equal(_np(q[i]), want_q) and np.array_equal(_np(s[i]), want_s)
    v = ops.dequantize_fp8(q, s, out_dtype=torch.float32)
    assert torch.equal(v, ops.dequantize_fp8(q, s.contiguous(), out_dtype=torch.float32))
    w = torch.randn(2, 3, 130, 144, generator=gen, device="cuda")
    q, s = ops.quantize_fp8(w, block_rows=128)
    assert s.shape == (2, 3, 2, 2)
    for i in range(6):
        want_q, want_s = ref.quantize(_np(w.view(6, 130, 144)[i]), 128)
        assert np.array_equal(_np(q.view(torch.uint8).view(6, 130, 144)[i].view(torch.float8_e4m3fn)), want_q)
        assert np.array_equal(_np(s.view(6, 2, 2)[i]), want_s)
    v = ops.dequantize_fp8(q, s, block_rows=128, out_dtype=torch.float32)
    each = s.repeat_interleave(128, 2)[:, :, :130].repeat_interleave(128, 3)[..., :144]
    assert torch.equal(v, q.float() * each)
    # one scale for every row, as a broadcast view
    one = torch.tensor([[0.5]], device="cuda").expand(3, 1)
    z = torch.randn(3, 64, generator=gen, device="cuda").to(torch.float8_e4m3fn)
    assert torch.equal(ops.dequantize_fp8(z, one, out_dtype=torch.float32), z.float() * 0.5)


def test_quantize_positions():
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(37, 272, generator=gen, device="cuda").to(torch.bfloat16)
    pos = torch.randperm(74, generator=gen, device="cuda").int().view(37, 2)
    q, s = ops.quantize_fp8(x, positions=pos)
    q0, s0 = ops.quantize_fp8(x)
    for j in range(2):
        assert torch.equal(_bytes(q)[pos[:, j].long()], _bytes(q0)) and torch.equal(s[pos[:, j].long()], s0)
    # places outside the output are skipped, nothing else is written
    sentinel = torch.full((8, 32), 7, dtype=torch.uint8, device="cuda")
    scales = torch.full((1, 8), 9.0, device="cuda")
    places = torch.tensor([3, -1, 99, 5], dtype=torch.int32, device="cuda")
    y = torch.randn(4, 32, generator=gen, device="cuda")
    capi.call("lmoe_quantize_fp8", y.data_ptr(), 2, 4, 32, 32, 0, places.data_ptr(), 1, 8, sentinel.data_ptr(),
              scales.data_ptr(), 8, capi.stream_handle())
    assert (sentinel[[0, 1, 2, 4, 6, 7]] == 7).all() and (scales[0, [0, 1, 2, 4, 6, 7]] == 9).all()
    assert (scales[0, [3, 5]] != 9).all()


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_more_than_2_to_the_31_values(block_rows):
    """The first rows, those around the 2^31st value and the last ones are what they are by themselves."""
    K = 4096
    rows = 2 ** 31 // K + 1024
    x = torch.empty(rows, K, dtype=torch.bfloat16, device="cuda").normal_()
    q, s = ops.quantize_fp8(x, block_rows=block_rows)
    v = ops.dequantize_fp8(q, s, block_rows=block_rows)
    for a in (0, rows - 1152, rows - 1024, rows - 128):
        part, scales = ops.quantize_fp8(x[a:a + 128], block_rows=block_rows)
        assert torch.equal(_bytes(q)[a:a + 128], _bytes(part))
        assert torch.equal(s[a // block_rows:(a + 128) // block_rows], scales)
        assert torch.equal(v[a:a + 128], ops.dequantize_fp8(part, scales, block_rows=block_rows))


def _bytes(q):
    return q.view(torch.uint8)


def test_quantize_empty_and_refusals():
    for shape in ((0, 64), (3, 0, 64), (0, 3, 64)):
        for b in (1, 128):
            q, s = ops.quantize_fp8(torch.zeros(shape, device="cuda"), block_rows=b)
            assert q.shape == shape and ops.dequantize_fp8(q, s, block_rows=b).shape == shape
    x = torch.zeros(4, 64, device="cuda")
    q, s = ops.quantize_fp8(x)
    for call, msg in (
            (lambda: ops.quantize_fp8(x[:, :40]), "multiple of 16"),
            (lambda: ops.quantize_fp8(x.double()), "bf16, fp16 or fp32"),
            (lambda: ops.quantize_fp8(x[0]), "rows, K"),
            (lambda: ops.quantize_fp8(x, block_rows=64), "block_rows"),
            (lambda: ops.quantize_fp8(x, block_rows=128, positions=torch.zeros(4, 1, dtype=torch.int32, device="cuda")),
             "positions"),
            (lambda: ops.quantize_fp8(x, positions=torch.zeros(4, 1, device="cuda")), "int32"),
            (lambda: ops.quantize_fp8(x, positions=torch.zeros(3, dtype=torch.int32, device="cuda")), "same number"),
            (lambda: ops.dequantize_fp8(q, s[:3]), "shape mismatch"),
            (lambda: ops.dequantize_fp8(q, s, block_rows=128), "shape mismatch"),
            (lambda: ops.dequantize_fp8(_bytes(q), s), "float8_e4m3fn"),
            (lambda: ops.dequantize_fp8(q, s.half()), "fp32"),
            (lambda: ops.dequantize_fp8(q, s, out_dtype=torch.float64), "out_dtype"),
            (lambda: ops.dequantize_fp8(q, s.cpu()), "CUDA")):
        with pytest.raises(RuntimeError, match=msg):
            call()


# --------------------------------------------------------------------------------- product
def _operands(R, E, N, K, swiglu, seed=0, std=0.05):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = ops.quantize_fp8(torch.randn(R, K, generator=gen, device="cuda"))
    w = [ops.quantize_fp8(torch.randn(E, N, K, generator=gen, device="cuda") * std, block_rows=128)
         for _ in range(1 + swiglu)]
    return x, w


def _want(x, w, off, K):
    """Output and its bound before the rounding to the output type, in 64 bits on the GPU."""
    qx, sx = x
    R = qx.shape[0]
    N = w[0][0].shape[1]
    KB = ref.blocks(K)
    out = torch.zeros(R, N, dtype=torch.float64, device="cuda")
    err = torch.zeros_like(out)
    rel = 128 * 2.0 ** -23 + (KB + 3) * 2.0 ** -24
    full = lambda q, s, b: q.double() * (s if b == 1 else s.repeat_interleave(128, 0)[:q.shape[0]]).double() \
        .repeat_interleave(128, 1)[:, :q.shape[1]]
    for e in range(len(off) - 1):
        a, b = off[e], off[e + 1]
        if a == b:
            continue
        xv = full(qx[a:b], sx[a:b], 1)
        y, m = [], []
        for q, s in w:
            wv = full(q[e], s[e], 128)
            y.append(xv @ wv.T)
            m.append(rel * (xv.abs() @ wv.abs().T))
        if len(w) == 1:
            out[a:b], err[a:b] = y[0], m[0]
        else:
            g, u = y
            act = g * torch.sigmoid(g)
            out[a:b] = act * u
            # |silu'| <= 1.1; exponential, division and products: 2^-20 of the value, and at least the last place
            # of the smallest normal number
            err[a:b] = 1.1 * m[0] * (u.abs() + m[1]) + act.abs() * m[1] + 2.0 ** -20 * out[a:b].abs() + 2.0 ** -125 * u.abs()
    return out, err


def _check_gemm(x, w, off, odt="bf16", i64=False, **kw):
    E = w[0][0].shape[0]
    K = x[0].shape[1]
    o = torch.tensor(off, dtype=torch.int64 if i64 else torch.int32, device="cuda")
    up = {} if len(w) == 1 else dict(weights_up=w[1][0], weight_scales_up=w[1][1])
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = ops.fp8_grouped_gemm(*x, *w[0], o, E, out_dtype=DT[odt], error=error, **up)
    want, err = _want(x, w, off, K)
    bound = err + HALF[odt] * (want.abs() + err) + (2.0 ** -25 if odt == "fp16" else 0.0)
    assert y.dtype == DT[odt] and y.shape == want.shape
    assert ((y.double() - want).abs() <= bound).all()
    inside = torch.zeros(y.shape[0], dtype=torch.bool)
    inside[off[0]:off[-1]] = True
    assert (y[~inside.cuda()] == 0).all()
    assert error.item() == 0
    return y


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("R,N,K,off", [
    (1, 8, 16, [0, 1]), (1, 1, 128, [0, 0, 1]), (5, 24, 272, [0, 2, 2, 5]), (40, 136, 144, [0, 40]),
    (33, 64, 128, [1, 7, 7, 30]), (257, 384, 1408, [0, 1, 200, 257]), (300, 129, 400, [0, 260, 290, 300]),
    (600, 520, 256, [3, 590]), (70, 1000, 2064, [0, 10, 70]), (129, 96, 4096, [0, 129]),
])
def test_gemm(R, N, K, off, swiglu):
    x, w = _operands(R, len(off) - 1, N, K, swiglu, seed=R)
    _check_gemm(x, w, off, i64=bool(R % 2))


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("odt", list(DT))
@pytest.mark.parametrize("N", [256, 250, 33])
def test_gemm_types_and_stores(odt, swiglu, N):
    x, w = _operands(150, 3, N, 320, swiglu, seed=N)
    _check_gemm(x, w, [4, 70, 70, 141], odt)


@pytest.mark.parametrize("swiglu", [False, True])
def test_gemm_many_tiles_a_pair(swiglu):
    """More tiles than CTA pairs, so that every ring wraps, of both widths."""
    x, w = _operands(1500, 9, 1400, 640, swiglu, seed=3)
    _check_gemm(x, w, [0, 300, 301, 301, 600, 900, 1156, 1157, 1413, 1500])
    x, w = _operands(12, 9, 2700, 1040, swiglu, seed=4)
    _check_gemm(x, w, [0, 1, 2, 3, 4, 5, 5, 7, 8, 12])


def test_gemm_scales_of_every_size():
    """A scale that is lost, swapped or taken from a neighbour changes the output by far more than its bound."""
    x, w = _operands(200, 2, 400, 1300 // 16 * 16, True, seed=5)
    gen = torch.Generator(device="cuda").manual_seed(6)
    spread = lambda s: torch.exp2(torch.randint(-20, 20, s.shape, generator=gen, device="cuda").float()) * \
        (1 + torch.rand(s.shape, generator=gen, device="cuda"))
    x = (x[0], spread(x[1]))
    w = [(w[0][0], spread(w[0][1]) * 1e-6), (w[1][0], spread(w[1][1]))]
    _check_gemm(x, w[:1], [0, 90, 200], "fp32")
    _check_gemm(x, w, [0, 90, 200], "fp32")


def test_gemm_long_sums_of_one_sign():
    K = 16384
    x = ops.quantize_fp8(0.5 + torch.rand(3, K, device="cuda"))
    w = [ops.quantize_fp8(0.5 + torch.rand(1, 40, K, device="cuda"), block_rows=128)]
    y = _check_gemm(x, w, [0, 3], "fp32")
    want, _ = _want(x, w, [0, 3], K)
    assert ((y.double() - want).abs() / want).max().item() < 5e-6


def test_gemm_values_that_are_not_finite():
    """NaN scales poison their rows, or their features, and nothing else."""
    x, w = _operands(60, 2, 300, 400, False, seed=8)
    base = _check_gemm(x, w, [0, 30, 60], "fp32")
    xs = x[1].clone()
    xs[7, 2] = float("nan")
    ws = w[0][1].clone()
    ws[1, 1, 0] = float("nan")
    o = torch.tensor([0, 30, 60], dtype=torch.int32, device="cuda")
    y = ops.fp8_grouped_gemm(x[0], xs, w[0][0], ws, o, 2, out_dtype=torch.float32)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[7] = True
    bad[30:, 128:256] = True
    assert torch.equal(torch.isnan(y), bad) and torch.equal(y[~bad], base[~bad])


def test_gemm_strides_and_alignment():
    gen = torch.Generator(device="cuda").manual_seed(9)
    x, w = _operands(50, 2, 200, 272, False, seed=9)
    want = _check_gemm(x, w, [0, 20, 50])
    o = torch.tensor([0, 20, 50], dtype=torch.int32, device="cuda")
    for xs in (x[1].contiguous(), x[1].clone(), torch.cat([x[1], x[1]], 1)[:, :3]):
        assert torch.equal(ops.fp8_grouped_gemm(x[0], xs, *w[0], o, 2), want)
    odd = torch.empty(50 * 272 + 1, dtype=torch.uint8, device="cuda")[1:].view(50, 272)
    odd.copy_(_bytes(x[0]))
    wide = torch.zeros(50, 300, dtype=torch.uint8, device="cuda")
    wide[:, 5:277] = _bytes(x[0])
    for q in (odd, wide[:, 5:277]):
        assert torch.equal(ops.fp8_grouped_gemm(q.view(torch.float8_e4m3fn), x[1], *w[0], o, 2), want)
    ws = torch.zeros(2, 3, 4, device="cuda")
    ws[:, :2, :3] = w[0][1]
    assert torch.equal(ops.fp8_grouped_gemm(*x, w[0][0], ws[:, :2, :3], o, 2), want)
    one = torch.full((1, 1), 0.5, device="cuda").expand(50, 3)   # one scale for everything
    got = ops.fp8_grouped_gemm(x[0], one, *w[0], o, 2)
    assert torch.equal(got, ops.fp8_grouped_gemm(x[0], one.contiguous(), *w[0], o, 2))
    more = torch.randn(5, 200, 272, generator=gen, device="cuda")
    q, s = ops.quantize_fp8(more, block_rows=128)
    _bytes(q)[:2] = _bytes(w[0][0])
    s[:2] = w[0][1]
    assert torch.equal(ops.fp8_grouped_gemm(*x, q, s, o, 2), want)   # experts behind the last are not read


@pytest.mark.parametrize("off", [[0, 9, 5, 20], [0, 5, 9, 21], [-1, 5, 9, 20]])
def test_gemm_bad_offsets(off):
    """Every row counts as outside, the error word says so, nothing outside the output is touched."""
    x, w = _operands(20, 3, 40, 64, False)
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = ops.fp8_grouped_gemm(*x, *w[0], torch.tensor(off, dtype=torch.int32, device="cuda"), 3, error=error)
    assert (y == 0).all() and error.item() != 0


def test_gemm_replayed_on_its_stream_with_new_values():
    x, w = _operands(100, 2, 300, 528, True, seed=11)
    o = torch.tensor([0, 40, 100], dtype=torch.int32, device="cuda")
    call = lambda: ops.fp8_grouped_gemm(*x, *w[0], o, 2, weights_up=w[1][0], weight_scales_up=w[1][1])
    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = call()
    g.replay()
    assert torch.equal(y, first)
    o.copy_(torch.tensor([0, 70, 90], dtype=torch.int32))
    x[1].mul_(1.5)
    g.replay()
    assert torch.equal(y, call())


def test_gemm_calls_at_once():
    """Two streams, each its own calls, give what one gives."""
    x, w = _operands(300, 3, 700, 1040, False, seed=12)
    o = torch.tensor([0, 100, 120, 300], dtype=torch.int32, device="cuda")
    want = ops.fp8_grouped_gemm(*x, *w[0], o, 3)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(ops.fp8_grouped_gemm(*x, *w[0], o, 3))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in outs)


def test_gemm_under_a_limit_of_ctas():
    x, w = _operands(300, 3, 700, 272, True, seed=13)
    off = [0, 100, 120, 300]
    want = _check_gemm(x, w, off)
    capi.lib().lmoe_set_gemm_sm_limit(5)
    try:
        got = _check_gemm(x, w, off)
    finally:
        capi.lib().lmoe_set_gemm_sm_limit(0)
    assert torch.equal(got, want)


@pytest.mark.parametrize("experts", [1, 250])
def test_gemm_more_than_2_to_the_31_codes(experts):
    """Of rows (tiles of rows, or with many experts the other kernel's limit of rows), and of weights."""
    K = 16384
    R = 2 ** 31 // K + 200 if experts == 1 else 64
    N = 40 if experts == 1 else 2 ** 31 // K // 249
    q = torch.randint(0, 2 ** 32, (R, K // 4), device="cuda").to(torch.int32).view(torch.uint8)
    q[(q & 0x7f) == 0x7f] = 0   # NaN
    q = q.view(torch.float8_e4m3fn)
    xs = torch.rand(K // 128, R, device="cuda").t()
    w = torch.randint(0, 2 ** 32, (experts, N, K // 4), device="cuda").to(torch.int32).view(torch.uint8)
    w[(w & 0x7f) == 0x7f] = 0
    w = w.view(torch.float8_e4m3fn)
    ws = torch.rand(experts, -(-N // 128), K // 128, device="cuda")
    assert max(q.numel(), w.numel()) > 2 ** 31
    off = torch.zeros(experts + 1, dtype=torch.int64, device="cuda")
    off[-1] = R                 # the last expert's
    y = ops.fp8_grouped_gemm(q, xs, w, ws, off, experts, out_dtype=torch.float32)
    for a, b in ((0, 64), (R - 64, R)):
        few = torch.tensor([0, b - a], dtype=torch.int64, device="cuda")
        want = ops.fp8_grouped_gemm(q[a:b], xs[a:b], w[-1:], ws[-1:], few, 1, out_dtype=torch.float32)
        assert torch.isfinite(want).all() and torch.equal(y[a:b], want)


def test_gemm_empty_and_refusals():
    x, w = _operands(4, 2, 24, 64, True)
    (q, s), (u, t) = w
    o = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    assert ops.fp8_grouped_gemm(x[0][:0], x[1][:0], q, s, torch.zeros_like(o), 2).shape == (0, 24)
    bad = (
        (lambda: ops.fp8_grouped_gemm(x[0], x[1][:3], q, s, o, 2), "scales shape"),
        (lambda: ops.fp8_grouped_gemm(x[0], x[1], q, s[:, :, :0], o, 2), "scales shape"),
        (lambda: ops.fp8_grouped_gemm(x[0], x[1], q[:, :, :48], s, o, 2), "shape mismatch"),
        (lambda: ops.fp8_grouped_gemm(x[0], x[1], q, s, o, 3), "shape mismatch|num_experts"),
        (lambda: ops.fp8_grouped_gemm(x[0], x[1], q, s, o[:2], 2), "expert_offsets"),
        (lambda: ops.fp8_grouped_gemm(x[0], x[1], q, s, o, 2, weights_up=u), "belong together"),
        (lambda: ops.fp8_grouped_gemm(x[0], x[1], q, s, o, 2, weights_up=u[:, :16], weight_scales_up=t), "mismatch"),
        (lambda: ops.fp8_grouped_gemm(x[0], x[1], q, s, o, 2, out_dtype=torch.float64), "out_dtype"),
        (lambda: ops.fp8_grouped_gemm(_bytes(x[0]), x[1], q, s, o, 2), "float8_e4m3fn"),
        (lambda: ops.fp8_grouped_gemm(x[0], x[1].half(), q, s, o, 2), "fp32"),
        (lambda: ops.fp8_grouped_gemm(x[0], x[1], q.cpu(), s, o, 2), "CUDA"),
        (lambda: ops.fp8_grouped_gemm(x[0], x[1], q, s, o, 2, error=torch.zeros(2, dtype=torch.int32, device="cuda")),
         "error"),
    )
    for call, msg in bad:
        with pytest.raises(RuntimeError, match=msg):
            call()
