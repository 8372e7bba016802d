"""The block-scaled 8-bit format in 64 bits (numpy), written from its definition."""
import numpy as np
import torch

BLOCK, TOP, LEAST = 128, 448.0, 2.0 ** -126
GRID = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()   # codes 0 .. 126


def blocks(n):
    return -(-n // BLOCK)


def scale(top, power_of_two=False):
    """Scale of blocks with these largest absolute values (NaN where they are not finite)."""
    with np.errstate(over="ignore", invalid="ignore"):
        s = np.maximum((np.asarray(top, np.float64) / TOP).astype(np.float32), np.float32(LEAST))
    if power_of_two:
        m, e = np.frexp(s)
        s = np.where(np.isfinite(s), np.ldexp(np.float32(1), np.where(m > 0.5, e, e - 1)), s)
    return np.where(np.isfinite(top), s, np.nan).astype(np.float32)


def nearest(t):
    """The E4M3 value nearest to t (64 bits), of two as near the one of the even code; at most 448."""
    a = np.abs(t)
    hi = np.clip(np.searchsorted(GRID, a), 1, 126)
    lo = hi - 1
    dl, dh = np.abs(a - GRID[lo]), np.abs(GRID[hi] - a)
    return np.copysign(np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), GRID[lo], GRID[hi]), t)


def quantize(x, block_rows=1, power_of_two=False):
    """x [rows, K] -> code values [rows, K] and scales [row blocks, column blocks] (fp32)."""
    x = np.asarray(x, np.float64)
    rows, K = x.shape
    q = np.zeros((rows, K))
    s = np.zeros((-(-rows // block_rows), blocks(K)), np.float32)
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            at = (slice(i * block_rows, (i + 1) * block_rows), slice(j * BLOCK, (j + 1) * BLOCK))
            s[i, j] = scale(np.abs(x[at]).max(), power_of_two)
            if np.isfinite(s[i, j]):
                q[at] = nearest(x[at] / np.float64(s[i, j]))
    return q, s


def spread(s, rows, K, block_rows=1):
    """Scales [.., row blocks, column blocks] as one factor per value [.., rows, K]."""
    s = np.asarray(s, np.float64)
    return np.repeat(np.repeat(s, block_rows, -2)[..., :rows, :], BLOCK, -1)[..., :K]


def values(q, s, block_rows=1):
    """What codes (as values) and scales stand for."""
    q = np.asarray(q, np.float64)
    return q * spread(s, q.shape[-2], q.shape[-1], block_rows)
