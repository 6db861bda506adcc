"""Plain 64-bit forms of the operators in optimized_transducer_amd/answering.py (numpy)."""
import math

import numpy as np

BLOCK = 128
# the non-negative finite e4m3 values in order; the parity of the index is that of the mantissa
E4M3 = np.array([(m / 8.0) * 2.0 ** -6 if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7)
                 for e in range(16) for m in range(8)][:127])


def to_e4m3(q):
    """Nearest e4m3 value of each |q| <= 448 * (1 + 2^-20), ties to the even mantissa."""
    a = np.abs(q.astype(np.float64))
    hi = np.searchsorted(E4M3, a).clip(0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - E4M3[lo], E4M3[hi] - a
    take_lo = (dl < dh) | ((dl == dh) & (lo % 2 == 0))
    return np.copysign(np.where(take_lo, E4M3[lo], E4M3[hi]), q)


def quantize_blocks(x, block_rows):
    """(values float64, scale float32) of x (rows, D) float32."""
    rows, D = x.shape
    nr, nc = -(-rows // block_rows), -(-D // BLOCK)
    scale = np.zeros((nr, nc), np.float32)
    values = np.zeros((rows, D), np.float64)
    for i in range(nr):
        for j in range(nc):
            at = np.s_[i * block_rows:(i + 1) * block_rows, j * BLOCK:(j + 1) * BLOCK]
            block = x[at]
            with np.errstate(all="ignore"):
                s = np.float32(np.float64(np.abs(block).max()) / 448.0)
                if s < np.float32(2.0 ** -126):
                    s = np.float32(2.0 ** -126)
                scale[i, j] = s
                if np.isfinite(s):
                    values[at] = to_e4m3(block / s)
                else:
                    values[at] = np.where(np.isfinite(block / s), 0.0, np.nan)
    return values, scale


def project(x, xs, w, ws, bias):
    """(logits, magnitude) in float64: the magnitude is the sum of the terms' absolute values."""
    a = x * np.repeat(xs.astype(np.float64), BLOCK, 1)[:, :x.shape[1]]
    b = w * np.repeat(np.repeat(ws.astype(np.float64), BLOCK, 1)[:, :w.shape[1]], BLOCK, 0)[:w.shape[0]]
    c = np.zeros(w.shape[0]) if bias is None else bias.astype(np.float64)
    return a @ b.T + c, np.abs(a) @ np.abs(b).T + np.abs(c)


def sample_row(x, u, temperature, top_k, top_p, min_p):
    """(symbol, log_prob) of one row, entry by entry in the order of the definition."""
    x = x.astype(np.float64) + 0.0
    V = len(x)
    m = x.max() if not np.isnan(x).any() else math.nan
    if not math.isfinite(m) or math.isnan(u):
        return -1, -math.inf
    if not temperature > 0:
        return int(np.argmax(x)), 0.0
    with np.errstate(all="ignore"):
        z = (x - m) / np.float64(np.float32(temperature))
    z[np.isneginf(x)] = -math.inf
    w = np.exp(z)
    order = np.lexsort((np.arange(V), -x))
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        ws = w[order]
        run = np.cumsum(ws)
        before = np.concatenate([[0.0], run[:-1]])
        n = max(1, int((before < np.float64(np.float32(top_p)) * run[-1]).sum()))
        order = order[:n]
    if min_p > 0:
        order = order[w[order] >= min(np.float64(np.float32(min_p)), 1.0)]
    kept = np.zeros(V)
    kept[order] = w[order]
    run = np.cumsum(kept)
    hits = np.nonzero((run > np.float64(np.float32(u)) * run[-1]) & (kept > 0))[0]
    s = int(hits[0]) if len(hits) else int(np.nonzero(kept)[0][-1])
    return s, float(z[s] - math.log(run[-1]))


def sample(x, u, temperature, top_k, top_p, min_p):
    rows = x.shape[0]
    t, k, p, m = (np.broadcast_to(np.asarray(v), (rows,)) for v in (temperature, top_k, top_p, min_p))
    out = [sample_row(x[r], float(u[r]), float(t[r]), int(k[r]), float(p[r]), float(m[r])) for r in range(rows)]
    return np.array([s for s, _ in out], np.int32), np.array([lp for _, lp in out])
