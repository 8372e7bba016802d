"""CPU tests of the 8-bit floating-point entry points: the reference itself, sizes and refusals, before
any GPU work."""
import ctypes

import numpy as np
import pytest
import torch

import fp8_reference as ref
from light_moe_b200 import capi, ops

OK, INVALID, UNSUPPORTED = capi.LMOE_OK, capi.LMOE_ERR_INVALID_ARG, capi.LMOE_ERR_UNSUPPORTED
BUF = (ctypes.c_uint8 * 4096)()
P = (ctypes.addressof(BUF) + 255) // 256 * 256   # an aligned host address: refused calls never read it


def test_reference_rounding():
    """Against torch's own conversion, which rounds to nearest even."""
    x = torch.linspace(-448, 448, 20001, dtype=torch.float64).float()
    x = torch.cat([x, x * 2.0 ** -9, torch.from_numpy(ref.GRID).float(),
                   torch.from_numpy((ref.GRID[1:] + ref.GRID[:-1]) / 2).float()])
    want = x.to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ref.nearest(x.double().numpy()), want)


def test_reference_scales():
    s = ref.scale(np.array([0.0, 448.0, 449.0, np.inf, np.nan, 1e-45, 3e38]), True)
    assert s[0] == s[5] == 2.0 ** -126 and s[1] == 1.0 and s[2] == 2.0 and np.isnan(s[3]) and np.isnan(s[4])
    assert np.log2(s[6]) % 1 == 0 and s[6] * 448.0 >= 3e38
    assert ref.scale(np.array([1.0]))[0] == np.float32(1.0) / np.float32(448.0)


def _rows(x=P, dtype=0, rows=4, K=64, ldx=64, p2=0, pos=None, copies=1, out_rows=4, q=P, s=P, pitch=4):
    return capi.lib().lmoe_quantize_fp8(x, dtype, rows, K, ldx, p2, pos, copies, out_rows, q, s, pitch, None)


@pytest.mark.parametrize("bad", [
    dict(K=2 ** 31 - 8192, ldx=2 ** 31), dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(K=40), dict(K=0),
    dict(ldx=63), dict(copies=2), dict(out_rows=5), dict(out_rows=-1), dict(pos=P, copies=0), dict(pitch=3), dict(x=None), dict(q=None),
    dict(s=None), dict(q=P + 8), dict(x=P + 1), dict(s=P + 2), dict(pos=P + 2),
])
def test_quantize_rows_refusals(bad):
    assert _rows(**bad) == INVALID


def _blocks(x=P, dtype=0, count=2, rows=4, K=64, p2=0, q=P, s=P):
    return capi.lib().lmoe_quantize_fp8_blocks(x, dtype, count, rows, K, p2, q, s, None)


@pytest.mark.parametrize("bad", [
    dict(K=2 ** 31 - 16), dict(rows=2 ** 31 - 16), dict(dtype=3), dict(count=-1), dict(rows=-1), dict(rows=2 ** 31),
    dict(K=24), dict(K=0), dict(x=None), dict(q=None), dict(s=None), dict(q=P + 4), dict(x=P + 1), dict(s=P + 1),
])
def test_quantize_blocks_refusals(bad):
    assert _blocks(**bad) == INVALID


def _deq(q=P, s=P, sm=4, sr=1, sb=4, count=1, rows=4, K=64, block=1, dtype=0, out=P):
    return capi.lib().lmoe_dequantize_fp8(q, s, sm, sr, sb, count, rows, K, block, dtype, out, None)


@pytest.mark.parametrize("bad", [
    dict(K=2 ** 31 - 16), dict(dtype=3), dict(block=2), dict(block=0), dict(count=-1), dict(rows=-1), dict(K=8), dict(K=0),
    dict(sm=-1), dict(sr=-1), dict(sb=-1), dict(q=None), dict(s=None), dict(out=None), dict(q=P + 1), dict(out=P + 8), dict(s=P + 2),
])
def test_dequantize_refusals(bad):
    assert _deq(**bad) == INVALID


def _gemm(xq=P, xs=P, pitch=4, R=4, K=64, wq=P, ws=P, uq=None, us=None, N=8, off=P, i64=0, E=2, odt=0, out=P):
    return capi.lib().lmoe_fp8_grouped_gemm(xq, xs, pitch, R, K, wq, ws, uq, us, N, off, i64, E, odt, out, None, None)


@pytest.mark.parametrize("bad", [
    dict(odt=3), dict(R=-1), dict(R=2 ** 31 - 1, pitch=2 ** 31), dict(N=0), dict(N=2 ** 30), dict(K=0), dict(K=40),
    dict(K=2 ** 31 - 16), dict(E=0), dict(uq=P), dict(us=P), dict(pitch=3), dict(xq=None), dict(xs=None),
    dict(wq=None), dict(ws=None), dict(off=None), dict(out=None), dict(xq=P + 8), dict(xs=P + 2), dict(wq=P + 1),
    dict(ws=P + 1), dict(uq=P + 8, us=P), dict(out=P + 1), dict(out=P + 2, odt=2), dict(off=P + 4, i64=1),
])
def test_gemm_refusals(bad):
    assert _gemm(**bad) == INVALID


def test_gemm_refuses_too_many_experts():
    assert _gemm(E=257) == UNSUPPORTED


def _few(x=P, dtype=0, T=4, d=128, gw=P, gb=None, E=4, k=2, S=0, w1=P, w3=P, w2=P, s1=None, s3=None, s2=None, F=64,
         y=P, ids=P, wts=P, ws=P, wsb=1 << 30):
    return capi.lib().lmoe_moe_layer_few_tokens(x, dtype, T, d, gw, gb, E, k, S, w1, w3, w2, s1, s3, s2, F, y, ids, wts,
                                                ws, wsb, None)


@pytest.mark.parametrize("bad", [
    dict(dtype=2), dict(dtype=-1), dict(T=17), dict(T=-1), dict(d=32), dict(d=96), dict(d=16448), dict(F=48), dict(F=0),
    dict(F=65568), dict(E=0), dict(E=257), dict(k=0), dict(k=5), dict(E=20, k=17), dict(S=-1), dict(S=17),
    dict(s1=P), dict(s3=P), dict(s1=P, s3=P), dict(x=None), dict(gw=None), dict(w1=None), dict(w3=None),
    dict(w2=None), dict(y=None), dict(ids=None), dict(wts=None), dict(x=P + 8), dict(gw=P + 8), dict(w1=P + 16),
    dict(w3=P + 16), dict(w2=P + 16), dict(gb=P + 2), dict(y=P + 1), dict(ids=P + 2), dict(wts=P + 2),
    dict(s1=P + 1, s3=P, s2=P),
])
def test_few_tokens_refusals(bad):
    assert _few(**bad) == INVALID


def test_few_tokens_workspace():
    size = capi.lib().lmoe_few_tokens_workspace_bytes
    for bad in ((17, 128, 64, 4, 2, 0), (-1, 128, 64, 4, 2, 0), (1, 100, 64, 4, 2, 0), (1, 128, 40, 4, 2, 0),
                (1, 128, 64, 257, 2, 0), (1, 128, 64, 4, 5, 0), (1, 128, 64, 4, 2, 17)):
        assert size(*bad) == 0
    one = size(1, 128, 64, 4, 2, 0)
    assert one > 0 and size(2, 128, 64, 4, 2, 0) > one
    assert _few(ws=None) == _few(wsb=size(4, 128, 64, 4, 2, 0) - 1) == _few(ws=P + 8) == capi.LMOE_ERR_WORKSPACE
    assert _few(T=0, ws=None) == OK


def test_empty_calls_need_no_gpu():
    assert _rows(rows=0, out_rows=0, pitch=0) == OK
    assert _blocks(count=0) == OK and _blocks(rows=0) == OK
    assert _deq(count=0) == OK and _deq(rows=0) == OK
    assert _gemm(R=0, pitch=0) == OK


def test_ops_refuse_host_tensors():
    x = torch.zeros(2, 64)
    q = x.to(torch.float8_e4m3fn)
    s = torch.ones(2, 1)
    for call in (lambda: ops.quantize_fp8(x), lambda: ops.dequantize_fp8(q, s),
                 lambda: ops.fp8_grouped_gemm(q, s, q[None], s[None, :1], torch.zeros(2, dtype=torch.int32), 1)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_layer_takes_the_few_token_kernels_only_for_their_sizes():
    """The module's limits are the library's."""
    from light_moe_b200 import fp8

    size = capi.lib().lmoe_few_tokens_workspace_bytes
    T, d, F, S = fp8.FEW_TOKENS, fp8.FEW_TOKENS_HIDDEN, fp8.FEW_TOKENS_FFN, fp8.FEW_TOKENS_SHARED
    for E, k in ((1, 1), (fp8.MOST_EXPERTS, 16)):
        assert size(T, d, F, E, k, S) > 0
    assert size(T, d, F + 32, 4, 2, S) == 0 and size(T, d, F, 4, 2, S + 1) == 0
    assert size(T, d, F, fp8.MOST_EXPERTS + 1, 2, S) == 0
