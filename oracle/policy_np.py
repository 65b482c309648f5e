"""Losses on chosen log-probabilities in float64 numpy, one row (or pair) at a time."""
import numpy as np


def row_log_prob(z, a):
    """(lp of class a, probabilities) of one row of logits; NaN for a class outside the row."""
    m = z.max()
    e = np.exp(z - m)
    s = e.sum()
    if not 0 <= a < len(z):
        return np.nan, e / s
    return (z[a] - m) - np.log(s), e / s


def log_probs(z, actions, ignore=-100):
    """lp per row (0 where ignored) of logits z [rows, V], and the rows' probabilities."""
    lp, probs = np.zeros(len(z)), np.zeros(z.shape)
    for n, a in enumerate(actions):
        if a != ignore:
            lp[n], probs[n] = row_log_prob(z[n], a)
    return lp, probs


def logit_gradient(probs, actions, slope, ignore=-100):
    """slope[n] * ([j == a] - p_j), 0 for an ignored row."""
    g = np.zeros(probs.shape)
    for n, a in enumerate(actions):
        if a == ignore:
            continue
        d = -probs[n]
        if 0 <= a < probs.shape[1]:
            d = d.copy()
            d[a] += 1.0
        g[n] = slope[n] * d
    return g


def policy_terms(lp, actions, old, adv, ref, low, high, kl, ignore=-100):
    """Per row: the loss term and its derivative by lp (0 where ignored)."""
    term, slope = np.zeros(len(lp)), np.zeros(len(lp))
    for n, a in enumerate(actions):
        if a == ignore:
            continue
        r = np.exp(lp[n] - old[n])
        clipped = min(max(r, 1 - low), 1 + high)
        if r * adv[n] <= clipped * adv[n]:
            term[n], slope[n] = -r * adv[n], -r * adv[n]
        else:
            term[n] = -clipped * adv[n]
        if kl:
            g = ref[n] - lp[n]
            term[n] += kl * (np.expm1(g) - g)
            slope[n] -= kl * np.expm1(g)
    return term, slope


def preference_terms(lp, actions, offsets, ref, beta, smoothing, ignore=-100):
    """Per pair: margin and term; per row: the term's derivative by lp."""
    pairs = (len(offsets) - 1) // 2
    gap = np.where(np.asarray(actions) == ignore, 0.0, lp - (0.0 if ref is None else ref))
    margin, term, slope = np.zeros(pairs), np.zeros(pairs), np.zeros(len(lp))
    for i in range(pairs):
        yes = slice(offsets[i], offsets[i + 1])
        no = slice(offsets[pairs + i], offsets[pairs + i + 1])
        h = beta * (gap[yes].sum() - gap[no].sum())
        margin[i] = h
        term[i] = (1 - smoothing) * np.logaddexp(0, -h) + smoothing * np.logaddexp(0, h)
        d = beta * (smoothing / (1 + np.exp(-h)) - (1 - smoothing) / (1 + np.exp(h)))
        slope[yes] += d
        slope[no] -= d
    return margin, term, slope
