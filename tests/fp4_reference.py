"""The microscaled 4-bit formats from their definition, in 64 bits (numpy), for the tests."""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = {"mxfp4": 32, "nvfp4": 16}


def e4m3_table():
    """Values of the E4M3 bytes 0..126 (positive, finite)."""
    b = np.arange(127)
    e, m = b >> 3, b & 7
    return np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e.astype(float) - 10))


def nearest_even(t, grid):
    """Index of the entry of the ascending grid nearest to t >= 0 (beyond the last: the last);
    of two as near, the even index."""
    t = np.minimum(t, grid[-1])
    hi = np.minimum(np.searchsorted(grid, t), len(grid) - 1)
    lo = np.maximum(hi - 1, 0)
    dl, dh = np.abs(t - grid[lo]), np.abs(grid[hi] - t)
    return np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)


def quantize(x, fmt, g=1.0):
    """x [rows, K] float64 -> (codes [rows, K] 0..15, scale bytes [rows, K / block])."""
    rows, K = x.shape
    b = BLOCK[fmt]
    xb = x.reshape(rows, K // b, b)
    bad = ~np.isfinite(xb).all(-1)
    xb = np.where(bad[..., None], 0.0, xb)
    top = np.abs(xb).max(-1)
    if fmt == "mxfp4":
        e = np.frexp(np.where(top > 0, top, 2.0 ** -200))[1] - 1 - 2
        e = np.clip(e, -127, 127)
        unit, byte = np.ldexp(1.0, e), e + 127
    else:
        byte = nearest_even(top / (6.0 * g), e4m3_table())
        unit = e4m3_table()[byte] * g
    t = np.where(unit[..., None] > 0, np.abs(xb) / np.where(unit > 0, unit, 1.0)[..., None], 0.0)
    code = nearest_even(t, E2M1)
    code = np.where(np.signbit(xb) & (unit[..., None] > 0), code + 8, code)
    byte = np.where(bad, 255 if fmt == "mxfp4" else 127, byte)
    code = np.where(bad[..., None], 0, code)
    return code.reshape(rows, K).astype(np.uint8), byte.astype(np.uint8)


def scale_values(s, fmt):
    if fmt == "mxfp4":
        return np.where(s == 255, np.nan, np.ldexp(1.0, s.astype(np.int64) - 127))
    return np.where(s == 127, np.nan, e4m3_table()[np.minimum(s, 126)])


def unpack(q):
    return np.stack([q & 15, q >> 4], -1).reshape(*q.shape[:-1], -1)


def values(q, s, fmt, g=1.0):
    """Packed codes [..., K/2] and scale bytes -> float64 values."""
    c = unpack(q)
    v = E2M1[c & 7] * np.where(c >> 3, -1.0, 1.0)
    return v * np.repeat(scale_values(s, fmt), BLOCK[fmt], -1) * g
