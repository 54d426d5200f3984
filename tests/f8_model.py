"""Rows and weights in 8 bits, in 64 bits and without the library: what e4m3 codes
stand for, and what the norm and the gated activation write."""
import numpy as np


def _table():
    v = np.arange(256)
    e, m = v >> 3 & 15, v & 7
    x = np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7.0), m * 2.0 ** -9)
    x[v & 127 == 127] = np.nan
    return np.where(v & 128, -x, x)


VALUES = _table()  # of the 256 codes


def codes_of(q):
    """The codes of q (f64, at most 448 in magnitude): the nearest, ties to the even
    code; NaN for NaN."""
    q = np.asarray(q, np.float64)
    grid = VALUES[:127]
    hi = np.clip(np.searchsorted(grid, np.abs(q)), 1, 126)
    lo = hi - 1
    below, above = np.abs(q) - grid[lo], grid[hi] - np.abs(q)
    code = np.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.isnan(q), 127, code)
    return (code | np.where(np.signbit(q) & ~np.isnan(q), 128, 0)).astype(np.uint8)


def blocks_of(t):
    """t [M, K] as [M, ceil(K/128), 128], filled up with zeros."""
    M, K = t.shape
    kb = -(-K // 128)
    b = np.zeros((M, kb, 128), t.dtype)
    b.reshape(M, kb * 128)[:, :K] = t
    return b


def quotients(t):
    """448 t / a of rows t [M, K] and their blocks' a [M, ceil(K/128)], in 64 bits;
    NaN where a block is not finite."""
    K = t.shape[1]
    b = blocks_of(np.asarray(t, np.float64))
    bad = ~np.isfinite(b).all(-1)
    a = np.where(bad, np.nan, np.abs(np.where(np.isfinite(b), b, 0)).max(-1))
    with np.errstate(invalid="ignore"):
        q = np.where(a[..., None] == 0, b, 448 * b / np.where(a == 0, 1, a)[..., None])
    q = np.where(bad[..., None], np.nan, q)
    return q.reshape(t.shape[0], b.shape[1] * 128)[:, :K], a


def norm(x, r, gain, eps):
    """(h, t, factor [M, 1]) of the norm: h as it is stored, t the f32 products."""
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        h = x if r is None else (x.astype(np.float32) + r.astype(np.float32)).astype(x.dtype)
        f = h.astype(np.float64)
        factor = 1 / np.sqrt((f * f).mean(1, keepdims=True) + np.float32(eps).astype(np.float64))
        return h, h.astype(np.float32) * gain.astype(np.float32), factor


def row_values(codes, scales):
    """What rows of codes [M, K] with scales [M, >= ceil(K/128)] stand for."""
    K = codes.shape[-1]
    s = np.repeat(scales[..., :-(-K // 128)].astype(np.float64), 128, -1)[..., :K]
    return VALUES[codes] * s


def weight_values(codes, scales):
    N, K = codes.shape[-2:]
    s = np.repeat(np.repeat(scales.astype(np.float64), 128, -2)[..., :N, :], 128, -1)[..., :K]
    return VALUES[codes] * s
