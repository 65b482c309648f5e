"""The gated linear recurrence and its gradients in float64, step by step, and how far a computation
that groups its steps otherwise may be from them."""
from __future__ import annotations

import numpy as np


def _walk(g, b, start):
    """h_t = g_t h_(t-1) + b_t along axis 1 and, in units of a rounding, its error: the term of step k
    in h_t is rounded at most 2 (t - k) + 16 times (a product and a sum for each step that it is
    carried over, one of each for each of at most seven joins of a scan, and itself)."""
    h, size, err = np.empty_like(b), np.abs(start), 16 * np.abs(start)
    errs = np.empty_like(b)
    now = start
    for t in range(b.shape[1]):
        gt, bt = g[:, t], b[:, t]
        with np.errstate(invalid="ignore"):
            now = np.where(gt == 0, bt, gt * now + bt)
            a = np.abs(gt)
            err = np.where(gt == 0, 0, a * (err + 2 * size)) + 16 * np.abs(bt)
            size = np.where(gt == 0, 0, a * size) + np.abs(bt)
        h[:, t], errs[:, t] = now, err
    return h, errs


def forward(x, g, state, mix):
    """(h, its error)"""
    with np.errstate(invalid="ignore"):
        b = np.where(g == 1, 0, (1 - g) * x) if mix else x
    return _walk(g, b, state)


def backward(x, g, state, gy, glast, mix):
    """((dx, error), (dgate, error), (dstate, error))"""
    h, eh = forward(x, g, state, mix)
    before = np.concatenate([state[:, None], h[:, :-1]], 1)
    eb = np.concatenate([0 * state[:, None], eh[:, :-1]], 1)
    # G_t = gy_t + g_(t+1) G_(t+1): the same walk from the end, the last step with the state's gradient
    after = np.concatenate([g[:, 1:], np.ones_like(g[:, :1])], 1)
    whole, ew = _walk(after[:, ::-1], gy[:, ::-1], glast)
    whole, ew = whole[:, ::-1], ew[:, ::-1]
    with np.errstate(invalid="ignore"):
        if mix:
            dx = np.where(g == 1, 0, (1 - g) * whole)
            edx = np.where(g == 1, 0, np.abs(1 - g) * ew) + 2 * np.abs(dx)
            base = before - x
        else:
            dx, edx, base = whole, ew, before
        dg = whole * base
        edg = np.abs(whole) * (eb + np.abs(base)) + np.abs(base) * ew + 2 * np.abs(dg)
        ds = np.where(g[:, 0] == 0, 0, g[:, 0] * whole[:, 0])
        eds = np.where(g[:, 0] == 0, 0, np.abs(g[:, 0]) * ew[:, 0]) + 2 * np.abs(ds)
    return (dx, edx), (dg, edg), (ds, eds)
