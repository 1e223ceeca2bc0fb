"""Plain 64-bit forms of the decode step's operators (numpy), for the tests: the draw from given
uniforms by its definition, and the codes, scales and product of the 8-bit head."""
from __future__ import annotations

import numpy as np

OK, INVALID, NAN = 0, -1, -2
NONE = 0xFFFFFFFF


def draw_row(x, temperature, top_k, top_p, min_p, u):
    """(status, token, prob, kept) of one row; x any float array (taken as it is, in 64 bits)."""
    x = np.asarray(x, np.float64)
    n = len(x)
    t = float(np.float32(temperature))
    bad = (INVALID, NONE, 0.0, 0)
    if not np.isfinite(t):
        return bad
    if t > 0 and (np.isnan(top_p) or not 0.0 <= min_p <= 1.0 or not 0.0 <= u < 1.0):
        return bad
    if np.isnan(x).any() or not np.isfinite(x.max()):
        return (NAN, NONE, 0.0, 0)
    if t <= 0:
        return (OK, int(np.argmax(x)), 1.0, 1)
    with np.errstate(over="ignore"):
        w = np.exp((x - x.max()) / t)
    order = np.argsort(-x, kind="stable")
    ranked = w[order]
    keep = int(np.isfinite(x).sum())
    if 0 < top_k < keep:
        keep = int(top_k)
    keep = min(keep, int((ranked[:keep] >= float(np.float32(min_p))).sum()))
    if 0 < top_p < 1:
        reach = np.cumsum(ranked)
        keep = min(keep, int((reach < float(np.float32(top_p)) * w.sum()).sum()) + 1)
    kept = np.zeros(n)
    kept[order[:keep]] = ranked[:keep]
    c = np.cumsum(kept)
    token = int(np.searchsorted(c, float(np.float32(u)) * c[-1], side="right"))
    return (OK, token, kept[token] / c[-1], keep)


def e4m3_values():
    """Value of every e4m3 code (0x7F and 0xFF are NaN)."""
    v = np.empty(256)
    for code in range(256):
        e, m = code >> 3 & 15, code & 7
        a = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v[code] = np.nan if code & 127 == 127 else -a if code & 128 else a
    return v


def blocks_of(a, rb, kb=128):
    """Largest magnitude of every rb x kb block of a 2-d array."""
    r = [np.abs(a[i:i + rb]).max(axis=0) for i in range(0, a.shape[0], rb)]
    return np.stack([[part[j:j + kb].max() for j in range(0, a.shape[1], kb)] for part in r])


def head(a, sa, w, sw):
    """The product in 64 bits and, beside each value, the sum of the magnitudes of its terms.
    a, w values of the codes; sa (rows, blocks), sw (ceil(n / 128), blocks)."""
    k = a.shape[1]
    x = a * np.repeat(sa.astype(np.float64), 128, axis=1)[:, :k]
    y = w * np.repeat(np.repeat(sw.astype(np.float64), 128, axis=1)[:, :k], 128, axis=0)[:w.shape[0]]
    return x @ y.T, np.abs(x) @ np.abs(y).T
