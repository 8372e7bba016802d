"""CPU tests of the 4-bit floating-point and gradient entry points: sizes and refusals, before
any GPU work."""
import ctypes

import numpy as np
import pytest
import torch

import fp4_reference as ref
from light_moe_b200 import capi, ops

INVALID, UNSUPPORTED, WORKSPACE = capi.LMOE_ERR_INVALID_ARG, capi.LMOE_ERR_UNSUPPORTED, capi.LMOE_ERR_WORKSPACE
BUF = (ctypes.c_uint8 * 4096)()
P = (ctypes.addressof(BUF) + 255) // 256 * 256   # an aligned host address: refused calls never read it


def test_scale_pitch():
    lib = capi.lib()
    assert lib.lmoe_fp4_scale_pitch(4096, capi.LMOE_FP4_MX) == 128
    assert lib.lmoe_fp4_scale_pitch(4096, capi.LMOE_FP4_NV) == 256
    assert lib.lmoe_fp4_scale_pitch(1408, capi.LMOE_FP4_MX) == 64     # 44 scales
    assert lib.lmoe_fp4_scale_pitch(1408, capi.LMOE_FP4_NV) == 96     # 88 scales
    assert lib.lmoe_fp4_scale_pitch(32, capi.LMOE_FP4_MX) == 32
    for K, f in ((0, 0), (-32, 0), (48, 1), (64, 2), (64, -1)):
        assert lib.lmoe_fp4_scale_pitch(K, f) == INVALID


def _quantize(x=P, dtype=0, rows=4, K=64, ldx=64, fmt=0, g=None, rps=1, pos=None, copies=1, out_rows=4, q=P, s=P):
    return capi.lib().lmoe_quantize_fp4(x, dtype, rows, K, ldx, fmt, g, rps, pos, copies, out_rows, q, s, None)


@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(rows=-1), dict(K=48), dict(K=0), dict(ldx=63), dict(fmt=2), dict(copies=2),
    dict(out_rows=5), dict(pos=P, copies=0), dict(g=P, rps=0), dict(x=None), dict(q=None), dict(s=None),
    dict(q=P + 4), dict(x=P + 1),
])
def test_quantize_refusals(bad):
    assert _quantize(**bad) == INVALID


def test_empty_calls_need_no_gpu():
    assert _quantize(rows=0, out_rows=0) == capi.LMOE_OK
    assert capi.lib().lmoe_dequantize_fp4(P, P, 32, 0, 64, 0, None, 1, P, None) == capi.LMOE_OK
    assert _gemm(R=0) == capi.LMOE_OK
    assert capi.lib().lmoe_grouped_gemm_dgrad(P, 0, 0, 8, P, 8, P, 0, 1, P, None, 0, None, None) == capi.LMOE_OK


@pytest.mark.parametrize("args", [
    (P, P, 1, 4, 64, 0, None, 1, P, None),        # pitch below the row's scales
    (P, P, 32, 4, 40, 0, None, 1, P, None),
    (P, P, 32, 4, 64, 7, None, 1, P, None),
    (P, P, 32, 4, 64, 1, P, 0, P, None),
    (P, P, 32, 4, 64, 0, None, 1, P + 8, None),
    (P + 4, P, 32, 4, 64, 0, None, 1, P, None),
    (None, P, 32, 4, 64, 0, None, 1, P, None),
])
def test_dequantize_refusals(args):
    assert capi.lib().lmoe_dequantize_fp4(*args) == INVALID


def _gemm(xq=P, xs=P, xp=32, R=4, K=64, wq=P, ws=P, uq=None, us=None, wp=32, N=8, fmt=0, off=P, i64=0, E=2, al=None,
          au=None, odt=0, out=P):
    return capi.lib().lmoe_fp4_grouped_gemm(xq, xs, xp, R, K, wq, ws, uq, us, wp, N, fmt, off, i64, E, al, au, odt,
                                            out, None, None)


@pytest.mark.parametrize("bad", [
    dict(fmt=2), dict(odt=3), dict(R=-1), dict(R=2 ** 31 - 1), dict(N=0), dict(K=0), dict(K=48), dict(E=0),
    dict(uq=P), dict(us=P), dict(xp=48), dict(wp=0), dict(xp=16), dict(K=2048, xp=32, wp=64), dict(xq=None),
    dict(xs=None), dict(wq=None), dict(ws=None), dict(off=None), dict(out=None), dict(xq=P + 8), dict(xs=P + 4),
    dict(wq=P + 1), dict(ws=P + 8), dict(out=P + 1), dict(out=P + 2, odt=2),
])
def test_gemm_refusals(bad):
    assert _gemm(**bad) == INVALID


def test_gemm_refuses_too_many_experts():
    assert _gemm(E=257) == UNSUPPORTED


def _dgrad(dy=P, dt=0, R=4, N=8, w=P, K=8, off=P, i64=0, E=2, dx=P, ws=None, wb=0):
    return capi.lib().lmoe_grouped_gemm_dgrad(dy, dt, R, N, w, K, off, i64, E, dx, ws, wb, None, None)


def _wgrad(dy=P, dt=0, R=4, N=8, x=P, K=8, off=P, i64=0, E=2, odt=0, dw=P, ws=None, wb=0):
    return capi.lib().lmoe_grouped_gemm_wgrad(dy, dt, R, N, x, K, off, i64, E, odt, dw, ws, wb, None, None)


@pytest.mark.parametrize("bad", [dict(dt=3), dict(R=-1), dict(N=0), dict(K=0), dict(E=0), dict(dy=None), dict(w=None),
                                 dict(off=None), dict(dx=None), dict(dy=P + 8), dict(w=P + 2), dict(dx=P + 1),
                                 dict(R=2 ** 31 - 1), dict(dt=2, dy=P + 2)])
def test_dgrad_refusals(bad):
    assert _dgrad(**bad) == INVALID


@pytest.mark.parametrize("bad", [dict(dt=3), dict(odt=1), dict(dt=1, odt=0), dict(dt=2, odt=0), dict(R=-1), dict(N=0),
                                 dict(K=0), dict(E=0), dict(dy=None), dict(x=None), dict(off=None), dict(dw=None),
                                 dict(x=P + 8), dict(odt=2, dw=P + 2)])
def test_wgrad_refusals(bad):
    assert _wgrad(**bad) == INVALID


def test_gradients_need_their_workspace():
    lib = capi.lib()
    size = lib.lmoe_grouped_gemm_grad_workspace_bytes
    assert size(0, 0, 100, 64, 64, 4) == 0                       # rows of multiples of 16 bytes: no copy
    assert size(0, 2, 100, 33, 31, 4) == 0                       # fp32 reads any row
    assert size(0, 0, 100, 33, 64, 4) == (100 * 40 * 2 + 255) // 256 * 256
    assert size(0, 1, 100, 64, 31, 4) == (4 * 64 * 32 * 2 + 255) // 256 * 256
    assert size(1, 0, 100, 64, 31, 4) == (100 * 32 * 2 + 255) // 256 * 256
    assert size(1, 0, -1, 64, 31, 4) == 0
    assert _dgrad(N=33) == WORKSPACE and _wgrad(K=31) == WORKSPACE
    assert _dgrad(N=33, ws=P, wb=16) == WORKSPACE
    assert _dgrad(N=33, ws=P + 8, wb=10 ** 6) == WORKSPACE
    assert _dgrad(E=300) == UNSUPPORTED and _wgrad(E=300) == UNSUPPORTED


def test_ops_refuse_host_tensors():
    x = torch.zeros(4, 64)
    q, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    off = torch.tensor([0, 4], dtype=torch.int32)
    for call in (lambda: ops.quantize_fp4(x, "mxfp4"), lambda: ops.dequantize_fp4(q, s, "mxfp4"),
                 lambda: ops.fp4_grouped_gemm(q, s, q[None], s[None], off, 1, "mxfp4"),
                 lambda: ops.grouped_gemm_dgrad(x, x[None], off, 1),
                 lambda: ops.grouped_gemm_wgrad(x, x, off, 1)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_reference_codes():
    """The oracle of the GPU tests on hand-worked blocks."""
    x = np.zeros((1, 32))
    x[0, :12] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.26, 7.9, 4.0, -1.0]   # top 7.9: scale 1
    c, s = ref.quantize(x, "mxfp4")
    assert s[0, 0] == 127 and c[0, :12].tolist() == [0, 2, 2, 4, 4, 6, 6, 7, 9, 7, 6, 10]
    c, s = ref.quantize(x / 16, "mxfp4")
    assert s[0, 0] == 123 and c[0, :12].tolist() == [0, 2, 2, 4, 4, 6, 6, 7, 9, 7, 6, 10]
    c, s = ref.quantize(x[:, :16] / 7.9 * 6, "nvfp4")
    assert s[0, 0] == 56 and c[0, 9] == 7                                              # byte 56 = 1.0
    assert ref.e4m3_table()[[1, 8, 56, 126]].tolist() == [2.0 ** -9, 2.0 ** -6, 1.0, 448.0]


@pytest.mark.parametrize("bad", [dict(xs=P + 16), dict(ws=P + 16), dict(uq=P, us=P + 16)])
def test_gemm_wants_scales_on_whole_sectors(bad):
    assert _gemm(**bad) == INVALID


TOP = 2 ** 31 - 1024   # sizes from here on leave no room for the index of the tile behind the last


def test_sizes_whose_tiles_pass_32_bits_are_refused():
    for K in (TOP, 2 ** 31 - 32):
        assert _gemm(K=K, xp=2 ** 27, wp=2 ** 27) == INVALID
    assert _gemm(N=TOP) == INVALID and _gemm(R=TOP) == INVALID
    for n in (TOP, 2 ** 31 - 1):
        assert _dgrad(N=n, ws=P, wb=2 ** 62) == INVALID and _dgrad(K=n, ws=P, wb=2 ** 62) == INVALID
        assert _wgrad(N=n, ws=P, wb=2 ** 62) == INVALID and _wgrad(K=n, ws=P, wb=2 ** 62) == INVALID
        for nk in ((n, 8), (8, n)):
            assert capi.lib().lmoe_grouped_gemm_any(P, 2, 4, nk[1], P, nk[0], P, 0, 2, P, None, 0, None, None) == INVALID


def test_no_workspace_for_sizes_that_are_refused():
    size = capi.lib().lmoe_grouped_gemm_grad_workspace_bytes
    for form in range(3):
        for dt in range(3):
            assert size(form, dt, 10, TOP, 33, 2) == 0 and size(form, dt, 10, 33, TOP, 2) == 0
            assert size(form, dt, TOP, 33, 33, 2) == 0
            assert size(form, dt, 10, TOP - 1, 33, 2) > 0
