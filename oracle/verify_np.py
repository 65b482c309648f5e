"""Verification of drafted tokens in float64, sequence by sequence."""
from __future__ import annotations

import numpy as np


def _softmax(z):
    """(probabilities, log-probabilities) of a row; NaN where it has none."""
    z = np.asarray(z, np.float64)
    m = np.max(z)
    if not np.isfinite(m):
        return np.full(z.shape, np.nan), np.full(z.shape, np.nan)
    s = np.sum(np.exp(z - m))
    with np.errstate(divide="ignore"):
        return np.exp(z - m) / s, z - m - np.log(s)


def _draw(w, r):
    sums = np.cumsum(w)
    above = np.nonzero((sums > r * sums[-1]) & (w > 0))[0]
    return int(above[0]) if len(above) else int(np.nonzero(w > 0)[0][-1])


def verify(logits, tokens, draft, uniforms, ignore=-100):
    """(tokens, accepted, log_probs) of arrays [S, K + 1, V], [S, K], [S, K, V] or None, [S, K + 1]."""
    S, K1, V = logits.shape
    K = K1 - 1
    out = np.full((S, K1), ignore, np.int64)
    lps, accepted = np.zeros((S, K1)), np.zeros(S, np.int64)
    u = np.asarray(uniforms, np.float64)
    for s in range(S):
        n = 0
        while True:
            p, lp = _softmax(logits[s, n])
            if n == K or tokens[s, n] == ignore:
                w = p
                break
            x = tokens[s, n]
            q = np.zeros(V) if draft is None else _softmax(draft[s, n])[0]
            inside = 0 <= x < V
            if draft is None:
                if inside:
                    q[x] = 1.0
                qx = 1.0
            else:
                qx = q[x] if inside else 0.0
            px = p[x] if inside else 0.0
            if u[s, n] * qx < px:
                out[s, n], lps[s, n] = x, lp[x]
                n += 1
                continue
            w = np.maximum(p - q, 0)          # NaN stays
            if not np.sum(w) > 0:
                w = p
            break
        accepted[s] = n
        if np.isnan(p).any():
            lps[s, n] = np.nan
        else:
            j = _draw(w, u[s, K])
            out[s, n], lps[s, n] = j, lp[j]
    return out, accepted, lps
