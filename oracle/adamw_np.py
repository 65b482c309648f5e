"""One AdamW step in float64, how far float32 may be from it, and moments in 8 bits."""
from __future__ import annotations

import numpy as np

U = 2.0**-24       # half a step of float32, relative


def scale_of(grads, max_norm):
    """min(1, max_norm / (norm + 1e-6)) over all gradients."""
    if not max_norm or max_norm <= 0:
        return 1.0
    norm = np.sqrt(sum(float(np.sum(np.square(np.asarray(g, np.float64)))) for g in grads))
    return min(1.0, max_norm / (norm + 1e-6))


def step(p, g, m, v, t, scale, lr, betas, eps, decay):
    """(p, m, v) after step number t, and the largest errors of a float32 computation of each: it
    rounds constants, products and sums by U (m: scale, its product, rest1, its product, the sum;
    v: scale and its product twice, the square, rest2, its product, the sum), takes a root and a
    reciprocal that are off by one unit (2 U) each, and rounds p twice."""
    p, g, m, v = (np.asarray(a, np.float64) for a in (p, g, m, v))
    b1, b2 = betas
    g = g * scale
    size_m = b1 * np.abs(m) + (1 - b1) * np.abs(g)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    d = np.sqrt(v) / np.sqrt(1 - b2**t) + eps
    size = lr / (1 - b1**t)
    with np.errstate(divide="ignore", invalid="ignore"):
        move = size * m / d
        err = 5 * U * size_m * size / d + 14 * U * np.abs(move)
    new = p * (1 - lr * decay) - move
    return ((new, 3 * U * np.maximum(np.abs(p), np.abs(new)) + err), (m, 5 * U * size_m),
            (v, 8 * U * v))


def step32(g, m, v, scale, betas):
    """The moments in float32, rounded product by product."""
    f = np.float32
    g, m, v = (np.asarray(a, f) for a in (g, m, v))
    g = g * f(scale)
    return m * f(betas[0]) + g * f(1 - betas[0]), v * f(betas[1]) + (g * g) * f(1 - betas[1])


def _blocks(a):
    a = np.asarray(a, np.float32).reshape(-1)
    return np.concatenate([a, np.zeros(-len(a) % 256, np.float32)]).reshape(-1, 256).astype(np.float64)


def _exponents(b, below):
    """Of each block's largest finite magnitude, less `below`, at least -126."""
    top = np.where(np.isfinite(b), np.abs(b), 0).max(1, keepdims=True)
    return np.maximum(np.frexp(np.maximum(top, 2.0**-1000))[1] - 1 - below, -126)


def _nearest(u, values):
    """The nearest of the sorted values, of two equally near the one at the even place."""
    hi = np.clip(np.searchsorted(values, u), 1, len(values) - 1)
    lo = hi - 1
    a, b = u - values[lo], values[hi] - u
    return np.where((a < b) | ((a == b) & (lo % 2 == 0)), lo, hi)


def _e4m3():
    """The values of e4m3 at or above 0, by their codes."""
    c = np.arange(127)
    e, f = c >> 3, c & 7
    return np.where(e == 0, f / 8 * 2.0**-6, (1 + f / 8) * 2.0**(e - 7.0))


def _e5m3():
    """0 and the values of codes 1..254 of exp_avg_sq."""
    c = np.arange(1, 255) + 770
    return np.concatenate([[0.0], (1 + (c & 7) / 8) * 2.0**((c >> 3) - 127.0)])


def _mixed(x):
    """The finalizer of MurmurHash3 (Appleby) of 32-bit numbers."""
    x = np.asarray(x, np.uint32)
    with np.errstate(over="ignore"):
        x = (x ^ (x >> np.uint32(16))) * np.uint32(0x85EBCA6B)
        x = (x ^ (x >> np.uint32(13))) * np.uint32(0xC2B2AE35)
    return x ^ (x >> np.uint32(16))


def words(t, n, first_tile=0):
    """The random words of step number t for the n elements of a tensor whose first tile of 2048 elements
    is number first_tile of the call."""
    key = _mixed(np.uint32(int(t) & 0xFFFFFFFF) ^ _mixed(np.uint32((int(t) >> 32) + 0x9E3779B9)))
    i = np.arange(n, dtype=np.uint64)
    tile, at = (i // 2048 + first_tile).astype(np.uint32), (i % 2048).astype(np.uint32)
    with np.errstate(over="ignore"):
        return _mixed(_mixed(tile + key) + at * np.uint32(0x9E3779B9))


def _at_random(u, values, fraction):
    """The place of u in the sorted values, of its two neighbours the upper one where the fraction of the
    way that is left to it is at most `fraction`."""
    lo = np.clip(np.searchsorted(values, u, side="right") - 1, 0, len(values) - 2)
    way = (u - values[lo]) / (values[lo + 1] - values[lo])
    # the kernel's 20 bits of it
    return lo + (np.floor(way * 2.0**20) / 2.0**20 + fraction >= 1)


def hold(m, v, random=None):
    """(codes of m, codes of v, exponents + 127) as 8 bits hold them: the nearest, or by random words of
    32 bits for each element, m by the lower half and v by the upper."""
    n = np.asarray(m).size
    if random is not None:
        random = np.concatenate([random, np.zeros(-n % 256, np.uint32)]).reshape(-1, 256)
        rm, rv = (((r & np.uint32(0xFFFF)) * 16.0 + 8) / 2.0**20 for r in (random, random >> np.uint32(16)))
        # (below 2^-6, the type's smallest normal number, the kernel's sum with it is rounded to float32)
        small = lambda u: np.where(u < 2.0**-6, (u + 2.0**-6).astype(np.float32).astype(np.float64) - 2.0**-6, u)
        place_m = lambda u: _at_random(small(u), _e4m3(), rm)
        place_v = lambda u: _at_random(u, _e5m3(), rv)
    else:
        place_m, place_v = (lambda u: _nearest(u, _e4m3())), (lambda u: _nearest(u, _e5m3()))
    bm, bv = _blocks(m), _blocks(v)
    km, kv = _exponents(bm, 7), _exponents(bv, 0)
    with np.errstate(invalid="ignore"):
        um, uv = bm * 2.0**-km, bv * 2.0**-kv
        cm = place_m(np.abs(np.where(np.isfinite(um), um, 0)))
        cm = np.where(np.signbit(um), cm | 0x80, cm)
        cm = np.where(np.isfinite(bm), cm, cm | 0x7F)
        fv = np.where(np.isfinite(uv), uv, 0)
        cv = np.where(fv > 0, np.maximum(place_v(fv), 1), 0)
        cv = np.where(np.isfinite(bv), cv, 255)
    powers = np.concatenate([km[:, 0], kv[:, 0]]) + 127
    return cm.reshape(-1)[:n].astype(np.uint8), cv.reshape(-1)[:n].astype(np.uint8), \
        powers.astype(np.uint8)


def values(cm, cv, powers):
    """What held moments stand for, in float64."""
    n = cm.size
    blocks = len(powers) // 2
    pad = lambda c: np.concatenate([c.reshape(-1), np.zeros(256 * blocks - n, np.uint8)]).reshape(blocks, 256)
    cm, cv = pad(cm), pad(cv)
    k = powers.astype(np.int64) - 127
    m = np.append(_e4m3(), np.nan)[cm & 127] * np.where(cm & 128, -1.0, 1.0) * 2.0**k[:blocks, None]
    v = np.append(_e5m3(), np.nan)[cv] * 2.0**k[blocks:, None]
    return m.reshape(-1)[:n], v.reshape(-1)[:n]
