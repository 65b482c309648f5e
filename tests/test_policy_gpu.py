"""Losses on chosen log-probabilities against the float64 oracle: values and gradients over types,
lengths, strides, masks, ragged sequences; graphs, streams, refusals."""
import concurrent.futures
import contextlib
import ctypes

import numpy as np
import pytest
import torch
import torch.utils.checkpoint

import compactlogic_amd as cl
from compactlogic_amd import _capi, policy, timing
from oracle import policy_np as P

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]
IGNORE = -100


def _unit(dtype):
    return 2.0**-53 if dtype == torch.float64 else 2.0**-24


def _sum_error(z, dtype):
    """Relative error of a row's sum of exponentials, and so the absolute one of lp: no chain of
    additions is longer than V / 256 + 32 (each rounds by a unit), an exponential is off by two
    units in the last place and by its argument's rounding, which weighs |x - m| exp(x - m) <= 1
    per term against a sum of at least 1, at most |x - m| <= spread of the finite logits."""
    fin = np.where(np.isfinite(z) & (np.abs(z) < 1e30), z, np.nan)
    spread = np.nanmax(fin) - np.nanmin(fin) if np.isfinite(fin).any() else 0.0
    return (z.shape[1] / 256 + 40 + min(spread, 100.0)) * _unit(dtype)


def _near(got, ref, err, dtype, half=None):
    """|got - ref| <= err + the rounding to `dtype` (half a step, and a subnormal's)."""
    got, ref = np.asarray(got, dtype=np.float64), np.asarray(ref, dtype=np.float64)
    info = torch.finfo(dtype)
    step = np.abs(ref) * (info.eps / 2) * 1.01 + info.smallest_normal * info.eps
    same = (got == ref) | (np.isnan(got) & np.isnan(ref))
    with np.errstate(invalid="ignore"):
        bad = ~(same | (np.abs(got - ref) <= err + step))
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], ref[bad][:5], np.max(err))


def _np(t):
    return t.detach().double().cpu().numpy()


def _wide(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


@pytest.fixture(params=[False, True], ids=["two passes", "one pass"])
def one_pass(request, monkeypatch):
    """The gradient out of the forward for every size that a workgroup holds, or for none."""
    def prefills(code, rows, cols):
        return request.param and code in (0, 3) and cols * (4 if code == 0 else 2) <= 131072
    monkeypatch.setattr(policy, "_prefills", prefills)
    return request.param


class Case:
    """Rows of logits and what the losses need beside them; ratios away from the borders of the
    clipped range (0.8, 1.28), so that rounding cannot change a row's side."""

    def __init__(self, rows, vocab, dtype, device, seed=0, scale=2.5, ignored=0.2):
        rng = np.random.default_rng(seed + 1000 * rows + vocab)
        z = torch.as_tensor(rng.standard_normal((rows, vocab)) * scale).to(dtype)
        self.dtype, self.wide = dtype, _wide(dtype)
        self.logits = z.to(device)
        self.z = _np(z)
        self.actions = rng.integers(0, vocab, rows)
        if rows > 2:
            self.actions[rng.random(rows) < ignored] = IGNORE
            self.actions[0] = vocab - 1
        self.lp, self.probs = P.log_probs(self.z, self.actions)
        ratio = rng.choice([0.4, 0.9, 1.0, 1.15, 1.7], rows)

        def wide(v):
            t = torch.as_tensor(v).to(self.wide)
            return t.to(device), _np(t)

        self.old_t, self.old = wide(self.lp - np.log(ratio))
        self.ref_t, self.ref = wide(self.lp + 0.3 * rng.standard_normal(rows))
        self.adv_t, self.adv = wide(rng.standard_normal(rows))
        self.act_t = torch.as_tensor(self.actions).to(device)
        self.err = _sum_error(self.z, dtype)

    def check_gradient(self, grad, slope, slope_err=0.0):
        """|[j = a] - p_j| <= 1: errors of the slope and of the probabilities pass as they are."""
        ref = P.logit_gradient(self.probs, self.actions, slope)
        err = (np.abs(slope) * 2 * self.err + slope_err)[:, None]
        assert grad.dtype == self.dtype
        _near(_np(grad), ref, np.where(np.isfinite(err), err, 0.0), self.dtype)


SIZES = [(1, 1), (1, 2), (3, 5), (128, 10), (33, 64), (9, 129), (5, 513), (7, 1000), (3, 2049),
         (4, 4099), (3, 8193), (2, 16385), (2, 33001), (3, 66000), (2, 131073), (1, 262147)]


@pytest.mark.parametrize("dtype", DTYPES)
def test_log_probs(device, dtype):
    for rows, vocab in SIZES:
        c = Case(rows, vocab, dtype, device)
        z = c.logits.requires_grad_()
        lp = cl.selected_log_probs(z, c.act_t)
        assert lp.dtype == c.wide and lp.shape == (rows,)
        _near(_np(lp), c.lp, c.err, c.wide)
        (g,) = torch.autograd.grad(lp, z, c.adv_t)
        c.check_gradient(g, c.adv)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("kl", [0.0, 0.05])
@pytest.mark.parametrize("dtype", DTYPES)
def test_policy_loss(device, one_pass, dtype, kl, reduction):
    for rows, vocab in SIZES:
        c = Case(rows, vocab, dtype, device)
        z = c.logits.requires_grad_()
        loss, lp = cl.policy_loss(z, c.act_t, c.old_t, c.adv_t,
                                  ref_log_probs=c.ref_t if kl else None, clip=(0.2, 0.28),
                                  kl_coef=kl, reduction=reduction, return_log_probs=True)
        term, slope = P.policy_terms(c.lp, c.actions, c.old, c.adv, c.ref, 0.2, 0.28, kl)
        counted = c.actions != IGNORE
        n = counted.sum()
        # |d term / d lp| <= 1.7 |A| + kl expm1(|g|); the terms are kept in the wide type
        bound = 1.8 * np.abs(c.adv) + kl * 5
        terr = bound * c.err + np.abs(term) * 2 * _unit(dtype)
        serr = 2 * bound * c.err
        _near(_np(lp), c.lp, c.err, c.wide)
        assert loss.dtype == c.wide
        if reduction == "none":
            up = np.random.default_rng(1).standard_normal(rows)
            ut = torch.as_tensor(up).to(c.wide).to(device)
            up = _np(ut)
            _near(_np(loss), term, terr, c.wide)
            (g,) = torch.autograd.grad(loss, z, ut)
            c.check_gradient(g, slope * up, serr * np.abs(up))
        else:
            div = n if reduction == "mean" else 1
            _near(_np(loss), term[counted].sum() / div, terr[counted].sum() / div, c.wide)
            for up in (1.0, 0.375):
                (g,) = torch.autograd.grad(loss * up, z, retain_graph=True)
                c.check_gradient(g, slope * up / div, serr * up / div)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("with_ref", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
def test_preference_loss(device, dtype, with_ref, reduction):
    for lengths, vocab, tail in [([1, 1], 200, 0), ([3, 1, 2, 5], 33, 0), ([0, 4, 3, 0], 1000, 2),
                                 ([300, 1, 2, 7, 31, 290], 129, 5), ([5, 2], 33001, 1),
                                 ([1] * 128, 10, 0)]:
        offsets = np.concatenate(([0], np.cumsum(lengths)))
        rows, pairs = int(offsets[-1]) + tail, len(lengths) // 2
        c = Case(rows, vocab, dtype, device, ignored=0.1)
        z = c.logits.requires_grad_()
        beta = 0.1 if with_ref else 0.02
        loss, margins = cl.preference_loss(
            z, c.act_t, torch.as_tensor(offsets).to(device),
            ref_log_probs=c.ref_t if with_ref else None, beta=beta, label_smoothing=0.1,
            reduction=reduction, return_margins=True)
        h, term, slope = P.preference_terms(c.lp, c.actions, offsets, c.ref if with_ref else None,
                                            beta, 0.1)
        seq = np.diff(offsets)
        herr = beta * (seq[:pairs] + seq[pairs:]) * c.err * 1.01
        assert margins.shape == (pairs,) and margins.dtype == c.wide
        _near(_np(margins), h, herr, c.wide)
        # |d term / d h| <= 1, |d slope / d h| <= beta / 4; both kept in the wide type
        serr = np.zeros(rows)
        for i in range(pairs):
            e = beta * herr[i] / 4 + 2 * beta * _unit(dtype)
            serr[offsets[i]:offsets[i + 1]] = e
            serr[offsets[pairs + i]:offsets[pairs + i + 1]] = e
        terr = herr + np.abs(term) * 2 * _unit(dtype)
        if reduction == "none":
            up = np.linspace(-1, 2, pairs)
            ut = torch.as_tensor(up).to(c.wide).to(device)
            _near(_np(loss), term, terr, c.wide)
            (g,) = torch.autograd.grad(loss, z, ut)
            row_up = np.zeros(rows)
            for i in range(pairs):
                row_up[offsets[i]:offsets[i + 1]] = _np(ut)[i]
                row_up[offsets[pairs + i]:offsets[pairs + i + 1]] = _np(ut)[i]
            c.check_gradient(g, slope * row_up, serr * np.abs(row_up)
                             + np.abs(slope * row_up) * 2 * _unit(dtype))
        else:
            div = pairs if reduction == "mean" else 1
            _near(_np(loss), term.sum() / div, terr.sum() / div, c.wide)
            for up in (1.0, 0.375):
                (g,) = torch.autograd.grad(loss * up, z, retain_graph=True)
                c.check_gradient(g, slope * up / div, serr * up / div)


@pytest.mark.parametrize("layout", ["padded", "offset", "transposed", "expanded", "batched"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [10, 301, 5003, 40001])
def test_layouts(device, one_pass, vocab, dtype, layout):
    """Strided, shifted and expanded logits against the oracle (a row is cut where its memory is
    aligned, so sums may be added in another order than for a contiguous copy)."""
    rows = 6
    c = Case(rows, vocab, dtype, device, ignored=0.0)
    z = c.logits
    if layout == "padded":
        t = torch.zeros((rows, vocab + 7), dtype=dtype, device=device)
        t[:, :vocab] = z
        x = t[:, :vocab]
    elif layout == "offset":
        t = torch.zeros(rows * vocab + 3, dtype=dtype, device=device)
        t[3:] = z.reshape(-1)
        x = t[3:].view(rows, vocab)
    elif layout == "transposed":
        x = z.t().contiguous().t()
    elif layout == "expanded":
        x = z[:1].expand(rows, vocab)
        c.z = np.repeat(c.z[:1], rows, 0)
        c.lp, c.probs = P.log_probs(c.z, c.actions)
        c.old_t, c.ref_t = [torch.as_tensor(c.lp + d).to(c.wide).to(device) for d in (0.05, -0.3)]
        c.old, c.ref = _np(c.old_t), _np(c.ref_t)
    else:
        x = z.view(2, 3, vocab)
    shape = x.shape[:-1]
    x = x.detach().requires_grad_()
    a, o, v, r = (t.view(shape) for t in (c.act_t, c.old_t, c.adv_t, c.ref_t))
    loss, lp = cl.policy_loss(x, a, o, v, r, kl_coef=0.1, reduction="sum", return_log_probs=True)
    assert lp.shape == shape
    _near(_np(lp).reshape(-1), c.lp, c.err, c.wide)
    term, slope = P.policy_terms(c.lp, c.actions, c.old, c.adv, c.ref, 0.2, 0.2, 0.1)
    bound = 1.8 * np.abs(c.adv) + 0.5
    _near(float(loss.detach()), term.sum(), (bound * c.err + np.abs(term) * 2 * _unit(dtype)).sum(),
          c.wide)
    c.check_gradient(torch.autograd.grad(loss, x)[0].reshape(rows, vocab), slope, 2 * bound * c.err)
    lp = cl.selected_log_probs(x, a)
    _near(_np(lp).reshape(-1), c.lp, c.err, c.wide)
    c.check_gradient(torch.autograd.grad(lp, x, v)[0].reshape(rows, vocab), c.adv)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [7, 300, 5001, 70001])
def test_masked_logits_and_rows(device, one_pass, vocab, dtype):
    """Masked classes (-inf, the type's lowest value), ignored rows full of NaN, rows with nothing
    left, actions that do not exist."""
    rows = 8
    c = Case(rows, vocab, dtype, device, ignored=0.0)
    z, a = c.logits.clone(), c.act_t.clone()
    a[:] = torch.arange(rows, device=device) % vocab
    low = torch.finfo(dtype).min
    z[0, 1:] = float("-inf")                # one class left: lp = 0, gradient 0
    z[1, 2:] = low                          # two classes left
    z[2] = float("nan")
    a[2] = IGNORE                           # does not count whatever it holds
    z[3] = float("-inf")                    # nothing left: NaN
    a[4] = vocab                            # no such class: NaN
    a[5] = -1
    z[6, 6 % vocab] = float("-inf")         # the chosen class is masked
    c.z, c.actions = _np(z), a.cpu().numpy()
    with np.errstate(invalid="ignore", divide="ignore"):
        c.lp, c.probs = P.log_probs(c.z, c.actions)
    c.err = _sum_error(c.z, dtype)
    c.old_t[2] = c.adv_t[2] = c.ref_t[2] = float("nan")
    z.requires_grad_()
    lp = cl.selected_log_probs(z, a)
    got = _np(lp)
    assert np.isnan(got[[3, 4, 5]]).all() and got[6] == -np.inf and got[2] == 0 and got[0] == 0
    _near(got, c.lp, c.err, c.wide)
    up = torch.ones_like(lp)
    (g,) = torch.autograd.grad(lp, z, up)
    g = _np(g)
    assert np.isnan(g[[3, 4, 5]]).all() and (g[2] == 0).all() and (g[0] == 0).all()
    ok = [0, 1, 2, 6, 7]
    ref = P.logit_gradient(c.probs, c.actions, np.ones(rows))
    _near(g[ok], ref[ok], 2 * c.err, dtype)
    # the losses: NaN rows make the loss NaN, not the gradient of the other rows
    loss = cl.policy_loss(z, a, c.old_t, c.adv_t, reduction="none")
    t = _np(loss)
    assert np.isnan(t[[3, 4, 5]]).all() and np.isfinite(t[ok]).all() and t[2] == 0
    total = cl.policy_loss(z, a, c.old_t, c.adv_t)
    (g,) = torch.autograd.grad(total, z)
    g = _np(g)
    assert np.isnan(float(total)) and np.isnan(g[[3, 4, 5]]).all() and np.isfinite(g[ok]).all()
    assert (g[2] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [7, 300, 5001, 20001, 70001])
def test_rows_of_the_lowest_value(device, one_pass, vocab, dtype):
    """A mask of the type's lowest value that leaves nothing, or one class of an ordinary or of the
    highest value: equal probabilities, or all of it for that class."""
    info = torch.finfo(dtype)
    z = torch.full((6, vocab), info.min, dtype=dtype, device=device)
    a = torch.tensor([0, vocab - 1, 2, 2, 2, 3], device=device)
    z[2, 2], z[3, 3], z[4, 2] = 1.5, -2.0, info.max
    z[5, :] = info.max
    z.requires_grad_()
    lp = cl.selected_log_probs(z, a)
    low = _np(z)[0, 0]
    zn = _np(z)
    zn = zn - zn.max(1, keepdims=True)       # in 64 bits these differences are finite
    lpn, probs = P.log_probs(zn, a.cpu().numpy())
    err = (vocab / 256 + 40) * _unit(dtype)
    want = _np(lp)
    ok = [0, 1, 2, 4, 5]
    _near(want[ok], lpn[ok], err, _wide(dtype))
    assert want[3] == -np.inf or want[3] <= low / 2      # beyond the wide type, or far down
    up = torch.ones(6, dtype=_wide(dtype), device=device)
    (g,) = torch.autograd.grad(lp, z, up)
    _near(_np(g), P.logit_gradient(probs, a.cpu().numpy(), np.ones(6)), 2 * err, dtype)
    old = torch.where(lp.detach().isinf(), 0, lp.detach())
    loss = cl.policy_loss(z, a, old, up, reduction="sum")
    (g,) = torch.autograd.grad(loss, z)
    slope = -np.exp(np.minimum(want - _np(old), 0.0))
    _near(_np(g), P.logit_gradient(probs, a.cpu().numpy(), slope), 4 * err, dtype)


def test_nothing_counts(device, one_pass):
    z = torch.randn(4, 9, device=device, requires_grad=True)
    a = torch.full((4,), IGNORE, device=device)
    f = torch.zeros(4, device=device)
    loss = cl.policy_loss(z, a, f, f)
    assert torch.isnan(loss)
    assert (torch.autograd.grad(loss, z)[0] == 0).all()
    assert float(cl.policy_loss(z, a, f, f, reduction="sum")) == 0
    off = torch.tensor([0, 2, 4], device=device)
    loss, h = cl.preference_loss(z, a, off, return_margins=True)
    assert float(h) == 0 and abs(float(loss) - np.log(2)) < 1e-6
    assert (torch.autograd.grad(loss, z)[0] == 0).all()
    # no rows, no pairs
    z0 = torch.empty(0, 9, device=device, requires_grad=True)
    a0, f0 = a[:0], f[:0]
    assert cl.selected_log_probs(z0, a0).shape == (0,)
    loss = cl.policy_loss(z0, a0, f0, f0)
    assert torch.isnan(loss) and torch.autograd.grad(loss, z0)[0].shape == (0, 9)
    assert float(cl.policy_loss(z0, a0, f0, f0, reduction="sum")) == 0
    assert cl.policy_loss(z0, a0, f0, f0, reduction="none").shape == (0,)
    loss, h = cl.preference_loss(z, a, off[:1], return_margins=True)
    assert torch.isnan(loss) and h.shape == (0,)
    assert (torch.autograd.grad(loss, z)[0] == 0).all()
    # a pair of empty sequences
    loss, h = cl.preference_loss(z0, a0, off[:1].expand(3), return_margins=True)
    assert float(h) == 0 and torch.autograd.grad(loss, z0)[0].shape == (0, 9)
    # another ignore_index
    b = torch.tensor([0, 3, 0, 5], device=device)
    lp = cl.selected_log_probs(z, b, ignore_index=0)
    ref = torch.log_softmax(z.detach().double(), 1)
    assert lp[0] == 0 and lp[2] == 0 and abs(float(lp[3]) - float(ref[3, 5])) < 1e-5


def test_bad_offsets_give_nan(device):
    """Offsets that decrease or leave the rows are read within the rows, and their pair is NaN."""
    c = Case(12, 20, torch.float32, device, ignored=0.0)
    for off in ([0, 5, 3, 8, 12], [0, 3, 6, 9, 13], [-1, 3, 6, 9, 12], [2**62, 3, 6, 9, 12],
                [0, 3, 6, 9, -2**62]):
        terms, h = cl.preference_loss(c.logits, c.act_t, torch.tensor(off, device=device),
                                      reduction="none", return_margins=True)
        bad = [any(not 0 <= off[q] <= off[q + 1] <= 12 for q in (i, 2 + i)) for i in range(2)]
        assert torch.isnan(terms).tolist() == bad and torch.isnan(h).tolist() == bad


def test_near_certain_policy(device):
    """1 - p of the chosen class, down to far below a unit of 1.  The row's sum 1 + 3 exp(-gap) is
    held in fp32: three additions next to 1 round by 2^-24 each, and so does the gradient's last
    product: 1 - p, which is known no better than the sum, is off by four of them."""
    for gap in (5.0, 12.0, 20.0, 40.0):
        z = torch.zeros(1, 4, device=device)
        z[0, 1] = gap
        z.requires_grad_()
        a = torch.ones(1, dtype=torch.int64, device=device)
        (g,) = torch.autograd.grad(cl.selected_log_probs(z, a).sum(), z)
        rest = -np.expm1(-np.log1p(3 * np.exp(-gap)))
        assert abs(float(g[0, 1]) - rest) <= 4 * 2.0**-24


def test_gradients_against_differences(device):
    """Central differences in float64 at 1e-6: cancellation leaves about 1e-10."""
    c = Case(6, 11, torch.float64, device, ignored=0.2)
    off = torch.tensor([0, 2, 3, 5, 6], device=device)
    fs = [lambda z: cl.selected_log_probs(z, c.act_t).mul(c.adv_t).sum(),
          lambda z: cl.policy_loss(z, c.act_t, c.old_t, c.adv_t, c.ref_t, kl_coef=0.3),
          lambda z: cl.preference_loss(z, c.act_t, off, c.ref_t, beta=0.7, label_smoothing=0.1)]
    for f in fs:
        z = c.logits.clone().requires_grad_()
        (g,) = torch.autograd.grad(f(z), z)
        d = torch.zeros_like(g)
        with torch.no_grad():
            for i in range(6):
                for j in range(11):
                    hi, lo = c.logits.clone(), c.logits.clone()
                    hi[i, j] += 1e-6
                    lo[i, j] -= 1e-6
                    d[i, j] = (f(hi) - f(lo)) / 2e-6
        assert float((g - d).abs().max()) < 1e-8


def test_second_backward_and_other_upstream(device, one_pass):
    """A retained graph gives the same gradient again, whatever was done with the first."""
    for dtype in (torch.float32, torch.bfloat16):
        for vocab in (10, 300, 3001, 8001, 20011, 33001):
            c = Case(40, vocab, dtype, device)
            z = c.logits.requires_grad_()
            loss = cl.policy_loss(z, c.act_t, c.old_t, c.adv_t)
            (g0,) = torch.autograd.grad(loss * 0, z, retain_graph=True)
            (g1,) = torch.autograd.grad(loss, z)
            assert not g0.any() and g1.any()
            (g2,) = torch.autograd.grad(cl.policy_loss(z, c.act_t, c.old_t, c.adv_t) * -2, z)
            assert torch.equal(g2, g1 * -2)          # a power of two: every rounding moves with it
            loss = cl.policy_loss(z, c.act_t, c.old_t, c.adv_t)
            (g1,) = torch.autograd.grad(loss, z, retain_graph=True)
            keep = g1.clone()
            (g2,) = torch.autograd.grad(loss * 0, z, retain_graph=True)
            (g3,) = torch.autograd.grad(loss, z, retain_graph=True)
            assert torch.equal(g1, keep) and torch.equal(g3, keep) and not g2.any()
            g1.zero_()
            (g4,) = torch.autograd.grad(loss, z)
            assert torch.equal(g4, keep)


def test_refusals(device):
    z = torch.zeros(3, 5, device=device)
    a = torch.zeros(3, dtype=torch.int64, device=device)
    f = torch.zeros(3, device=device)
    off = torch.tensor([0, 1, 2], device=device)
    with pytest.raises(RuntimeError, match="actions must be int64"):
        cl.selected_log_probs(z, a.int())
    with pytest.raises(RuntimeError, match="actions must be int64"):
        cl.selected_log_probs(z, a[:2])
    with pytest.raises(RuntimeError, match="same HIP device"):
        cl.selected_log_probs(z, a.cpu())
    with pytest.raises(RuntimeError, match="dtype"):
        cl.selected_log_probs(z.long(), a)
    with pytest.raises(RuntimeError, match="at least one class"):
        cl.selected_log_probs(z[:, :0], a)
    with pytest.raises(RuntimeError, match="old_log_probs must be"):
        cl.policy_loss(z, a, f[:2], f)
    with pytest.raises(RuntimeError, match="advantages must be"):
        cl.policy_loss(z, a, f, f.long())
    with pytest.raises(RuntimeError, match="detach"):
        cl.policy_loss(z, a, f.clone().requires_grad_(), f)
    with pytest.raises(RuntimeError, match="ref_log_probs must be"):
        cl.policy_loss(z, a, f, f, f.cpu())
    with pytest.raises(ValueError, match="clip"):
        cl.policy_loss(z, a, f, f, clip=-0.1)
    with pytest.raises(ValueError, match="kl_coef"):
        cl.policy_loss(z, a, f, f, kl_coef=0.1)
    with pytest.raises(ValueError, match="reduction"):
        cl.policy_loss(z, a, f, f, reduction="median")
    for bad in (off[:2], off.int(), off.cpu(), off.view(1, 3)):
        with pytest.raises(RuntimeError, match="offsets must be"):
            cl.preference_loss(z, a, bad)
    with pytest.raises(ValueError, match="label_smoothing"):
        cl.preference_loss(z, a, off, label_smoothing=1.5)
    with pytest.raises(RuntimeError, match="ragged batch"):
        cl.preference_loss(z[None], a[None], off)
    x = z.clone().requires_grad_()
    for f2 in (lambda y: cl.policy_loss(y, a, f, f + 1), lambda y: cl.preference_loss(y, a, off),
               lambda y: cl.selected_log_probs(y, a).sum()):
        with pytest.raises(RuntimeError, match="twice"):
            torch.autograd.grad(f2(x * x), x, create_graph=True)
    y = x * 1
    lp = cl.selected_log_probs(y, a)
    y += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        lp.sum().backward()


def test_half_precision_constants_are_widened(device):
    c = Case(20, 50, torch.bfloat16, device)
    old, adv = c.old_t.half(), c.adv_t.bfloat16()
    got = cl.policy_loss(c.logits, c.act_t, old, adv)
    assert torch.equal(got, cl.policy_loss(c.logits, c.act_t, old.float(), adv.float()))


def test_half_gradient_of_a_scaled_loss(device):
    """A mean over many rows in half precision: the gradient is formed from the scaled loss, not
    scaled after it was rounded to (or flushed below) half's smallest numbers."""
    c = Case(4096, 40, torch.float16, device)
    z = c.logits.requires_grad_()
    loss = cl.policy_loss(z, c.act_t, c.old_t, c.adv_t) * 65536.0
    (g,) = torch.autograd.grad(loss, z)
    term, slope = P.policy_terms(c.lp, c.actions, c.old, c.adv, c.ref, 0.2, 0.2, 0.0)
    n = (c.actions != IGNORE).sum()
    c.check_gradient(g, slope * 65536.0 / n, 2 * 1.8 * np.abs(c.adv) * c.err * 65536.0 / n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16])
@pytest.mark.parametrize("batch,feats,k,layout", [
    (1, 30, 10, "rows"), (63, 1200, 10, "columns"), (64, 12000, 10, "columns"),
    (130, 2001, 200, "columns"), (7, 25, 10, "rows"), (1024, 12000, 10, "rows"),
    (96, 777, 5, "strided"), (70, 1030, 513, "columns"), (5, 3, 7, "rows")])
def test_group_sum_methods(device, batch, feats, k, layout, dtype):
    """The three losses from a network's last activations against the oracle on scores summed in 64
    bits.  An fp32 partial sum adds at most feats / k + 8 numbers of up to 1, each addition off by a
    unit of the sum so far; the rest is fp64 until one rounding at the size of a difference.  (More
    than 512 classes take GroupSum's own fp32 scores, rounded at the size of the score.)"""
    rng = np.random.default_rng(batch + feats + k)
    tau = 2.0
    x = torch.as_tensor(rng.random((batch, feats))).to(dtype).to(device)
    xn = _np(x)
    if layout == "columns":
        x = x.t().contiguous().t()
    elif layout == "strided":
        x = torch.zeros((batch, 2 * feats), dtype=dtype, device=device)[:, ::2].copy_(x)
    x.requires_grad_()
    wide = _wide(dtype)
    gsz = -(-feats // k)
    padded = np.zeros((batch, gsz * k))
    padded[:, :feats] = xn
    z = padded.reshape(batch, k, gsz).sum(2) / tau
    actions = rng.integers(0, k, batch)
    actions[rng.random(batch) < 0.1] = IGNORE
    lp, probs = P.log_probs(z, actions)
    a = torch.as_tensor(actions).to(device)
    old = torch.as_tensor(lp - np.log(rng.choice([0.4, 0.9, 1.1, 1.7], batch))).to(wide).to(device)
    ref = torch.as_tensor(lp + 0.3 * rng.standard_normal(batch)).to(wide).to(device)
    adv = torch.as_tensor(rng.standard_normal(batch)).to(wide).to(device)
    spread = z.max() - z.min()
    unit = _unit(wide)
    score_err = (gsz + 8) * gsz * unit / tau + spread * unit
    if k > 512:
        score_err += np.abs(z).max() * unit
    err = 2 * score_err + _sum_error(z - z.max(1, keepdims=True), wide)
    gs = cl.GroupSum(k, tau)
    scale = np.repeat(np.eye(k), gsz, axis=1)[:, :feats] / tau      # d score / d x

    def check(grad, slope, serr):
        full = P.logit_gradient(probs, actions, slope)
        bound = ((np.abs(slope) * 2 * err + serr)[:, None] + np.abs(full) * 3 * unit) @ scale
        assert grad.dtype == dtype and grad.shape == (batch, feats)
        if layout == "columns" and batch > 1:
            assert grad.t().is_contiguous()
        _near(_np(grad), full @ scale, bound, dtype)

    got = gs.log_probs(x, a)
    assert got.dtype == wide
    _near(_np(got), lp, err, wide)
    check(torch.autograd.grad(got, x, adv)[0], _np(adv), 0.0)

    loss, lps = gs.policy_loss(x, a, old, adv, ref, clip=(0.2, 0.28), kl_coef=0.05,
                               return_log_probs=True, reduction="sum")
    term, slope = P.policy_terms(lp, actions, _np(old), _np(adv), _np(ref), 0.2, 0.28, 0.05)
    bound = 1.8 * np.abs(_np(adv)) + 0.25
    _near(_np(lps), lp, err, wide)
    _near(float(loss.detach()), term.sum(), (bound * err + np.abs(term) * 2 * unit).sum(), wide)
    check(torch.autograd.grad(loss, x)[0], slope, 2 * bound * err)

    pairs = batch // 2
    off = np.arange(2 * pairs + 1)
    loss, h = gs.preference_loss(x, a, torch.as_tensor(off).to(device), ref, beta=0.3,
                                 return_margins=True, reduction="sum")
    want, term, slope = P.preference_terms(lp, actions, off, _np(ref), 0.3, 0.0)
    _near(_np(h), want, 0.6 * err + 4 * unit, wide)
    _near(float(loss.detach()), term.sum(), (0.6 * err + 4 * unit) * max(pairs, 1)
          + np.abs(term).sum() * 2 * unit, wide)
    check(torch.autograd.grad(loss, x)[0], slope, 0.3 * 0.6 * err + 0.3 * 4 * unit)


def _centred_scores(x, k, tau):
    code = 0 if x.dtype == torch.float32 else 1
    need = ctypes.c_int64()
    _capi.call("cl_group_sum_centered_workspace_size", code, *x.shape, x.stride(0), k,
               ctypes.byref(need))
    ws = torch.empty(max(need.value, 1), dtype=torch.uint8, device=x.device)
    out = torch.empty((x.shape[0], k), dtype=x.dtype, device=x.device)
    _capi.call("cl_group_sum_centered_forward", code, x.data_ptr(), *x.shape, *x.stride(), k, tau,
               out.data_ptr(), ws.data_ptr(), need.value,
               torch.cuda.current_stream(x.device).cuda_stream)
    return out


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_group_sum_gradient_is_that_of_the_scores(device, dtype, reduction):
    """The fused backward gives what the losses' own gradient of the (centred) scores gives through
    GroupSum, bit by bit, in every layout and reduction."""
    batch, feats, k, tau = 96, 1201, 10, 3.0
    g = torch.Generator().manual_seed(5)
    base = torch.rand((batch, feats), generator=g, dtype=torch.float64).to(dtype).to(device)
    a = torch.randint(0, k, (batch,), generator=g).to(device)
    a[::9] = IGNORE
    old = (torch.randn(batch, generator=g) * 0.2 - 2.3).to(dtype).to(device)
    adv, ref = torch.randn(batch, generator=g).to(dtype).to(device), old + 0.1
    off = torch.tensor([0, 20, 40, 41, 60, 60, 90], device=device)
    gs = cl.GroupSum(k, tau)
    for x in (base.clone(), base.t().contiguous().t(), base[:, :1200:1].clone()):
        x.requires_grad_()
        seen = []
        scores = _centred_scores(x, k, tau).requires_grad_()
        up = torch.randn(batch if reduction == "none" else (), generator=g,
                         dtype=torch.float64).to(dtype).to(device)
        seen.append((gs.policy_loss(x, a, old, adv, ref, kl_coef=0.1, reduction=reduction),
                     cl.policy_loss(scores, a, old, adv, ref, kl_coef=0.1, reduction=reduction),
                     up))
        up = up[:3].contiguous() if reduction == "none" else up
        seen.append((gs.preference_loss(x, a, off, ref, beta=0.5, reduction=reduction),
                     cl.preference_loss(scores, a, off, ref, beta=0.5, reduction=reduction), up))
        seen.append((gs.log_probs(x, a), cl.selected_log_probs(scores, a), adv))
        for fused, apart, u in seen:
            assert torch.equal(fused, apart)
            (gx,) = torch.autograd.grad(fused, x, u)
            (gz,) = torch.autograd.grad(apart, scores, u)
            assert torch.equal(gx, torch.autograd.grad(gs(x), x, gz)[0])


def test_group_sum_methods_shapes(device):
    """Leading dimensions, non-finite activations, refusals."""
    gs = cl.GroupSum(5, 2.0)
    x = torch.rand(4, 3, 50, device=device)
    a = torch.randint(0, 5, (4, 3), device=device)
    lp = gs.log_probs(x, a)
    assert lp.shape == (4, 3)
    assert torch.equal(lp.view(-1), gs.log_probs(x.view(12, 50), a.view(-1)))
    y = x.view(12, 50).clone()
    y[3, 7], y[5, 8], y[6, 9] = float("nan"), float("inf"), float("-inf")
    bad = gs.log_probs(y, a.view(-1))
    assert torch.isnan(bad[3]) and torch.isnan(bad[5])
    ok = torch.ones(12, dtype=torch.bool)
    ok[[3, 5, 6]] = False
    assert torch.equal(bad.cpu()[ok], lp.view(-1).cpu()[ok])
    f = torch.zeros(12, device=device)
    with pytest.raises(RuntimeError, match="detach"):
        gs.policy_loss(y, a.view(-1), f.requires_grad_(), f)
    with pytest.raises(RuntimeError, match="dtype"):
        gs.log_probs(y.bfloat16(), a.view(-1))
    with pytest.raises(TypeError):
        gs.log_probs(cl.PackBitsTensor(y > 0.5, 64), a)
    with pytest.raises(RuntimeError, match="actions must be int64"):
        gs.log_probs(y, a)


def test_captured_policy_step(device, one_pass):
    """A policy step of a whole network (dropout, GroupSum, the clipped loss, Adam) captured once:
    every replay equals the eager step with the same mask."""
    torch.manual_seed(0)

    def build():
        torch.manual_seed(1)
        net = torch.nn.Sequential(cl.LogicLayer(60, 300, connections="original"),
                                  cl.Dropout(0.1, fill=0.5, seed=4), cl.LogicLayer(300, 300),
                                  cl.GroupSum(10, 3.0)).to(device)
        return net, cl.FusedAdam(net.parameters(), lr=0.01)

    x = (torch.rand(128, 60, device=device) < 0.4).float()
    a = torch.randint(0, 10, (128,), device=device)
    adv = torch.randn(128, device=device)
    net, opt = build()
    with torch.no_grad():
        old = net[3].log_probs(net[:3](x), a)
        ref = old + 0.1 * torch.randn(128, device=device)

    def step(net, opt):
        opt.zero_grad(set_to_none=True)
        loss, lp = net[3].policy_loss(net[:3](x), a, old, adv, ref_log_probs=ref, kl_coef=0.1,
                                      return_log_probs=True)
        loss.backward()
        opt.step()
        return loss.detach(), lp

    net, opt = build()
    eager = []
    for _ in range(6):
        loss, lp = step(net, opt)
        eager.append((loss.clone(), lp.clone(), [p.detach().clone() for p in net.parameters()]))
    net, opt = build()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(net, opt)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, lp = step(net, opt)
    for k in range(2, 6):
        junk = torch.randn(1000, device=device).sum()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = eager[k]
        assert torch.equal(loss, want[0]) and torch.equal(lp, want[1]), f"replay {k}"
        for p, w in zip(net.parameters(), want[2]):
            assert torch.equal(p, w), f"replay {k}"
        del junk


def test_policy_and_reference_under_one_mask(device):
    """As they are used together: a network with dropout records its log-probabilities under the
    masks of a step, and a later evaluation under the same masks has ratios of 1: the loss is minus
    the mean advantage, the margins against itself are 0, to rounding; other masks give others."""
    torch.manual_seed(2)
    layers = [cl.LogicLayer(60, 400, connections="original"), cl.LogicLayer(400, 400)]
    net = torch.nn.Sequential(*layers).to(device)
    head = cl.GroupSum(10, 3.0)
    x = (torch.rand(128, 60, device=device) < 0.4).float()
    a = torch.randint(0, 10, (128,), device=device)
    adv = torch.randn(128, device=device)

    def body(offset):
        return net[1](cl.dropout(net[0](x), 0.2, 77, offset, fill=0.5))

    with torch.no_grad():
        old = head.log_probs(body(3), a)
        other = head.log_probs(body(4), a)
    assert not torch.equal(old, other)
    loss, lp = head.policy_loss(body(3), a, old, adv, ref_log_probs=old, kl_coef=0.1,
                                return_log_probs=True)
    assert torch.equal(lp, old)
    # the recorded log-probabilities are rounded once, what the losses compare them with is not
    step = 2.0**-24 * float(old.abs().max())
    assert abs(float(loss.detach()) + float(adv.double().mean())) \
        <= float(adv.abs().mean()) * (step + 2.0**-22)
    loss.backward()
    assert all(p.grad.abs().sum() > 0 for p in net.parameters())
    off = torch.arange(0, 129, 2, device=device)[:65]
    loss, h = head.preference_loss(body(3), a, off, ref_log_probs=old, return_margins=True)
    assert float(h.abs().max()) <= 0.1 * 2 * 2 * step      # two sequences of two rows
    assert abs(float(loss.detach()) - np.log(2)) <= 0.1 * 2 * step + 2.0**-24
    _, h = head.preference_loss(body(3), a, off, ref_log_probs=other, return_margins=True)
    assert float(h.abs().max()) > 0.01


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [10, 3001, 70001])
def test_captured_losses(device, one_pass, dtype, vocab):
    """Each loss with its gradient captured; replays on new inputs equal the eager calls."""
    rows = 24
    off = torch.tensor([0, 5, 9, 16, 22], device=device)
    cases = [Case(rows, vocab, dtype, device, seed=s) for s in range(3)]
    c0 = cases[0]
    fs = [lambda z, c: cl.selected_log_probs(z, c.act_t).sum(),
          lambda z, c: cl.policy_loss(z, c.act_t, c.old_t, c.adv_t, c.ref_t, kl_coef=0.1),
          lambda z, c: cl.policy_loss(z, c.act_t, c.old_t, c.adv_t, reduction="sum") * 0.5,
          lambda z, c: cl.preference_loss(z, c.act_t, off, c.ref_t)]
    for f in fs:
        want = []
        for c in cases:
            z = c.logits.clone().requires_grad_()
            loss = f(z, c)
            want.append((loss.detach().clone(), torch.autograd.grad(loss, z)[0]))
            del loss, z
        static = Case(rows, vocab, dtype, device, seed=0)
        z = static.logits.clone().requires_grad_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            loss = f(z, static)
            torch.autograd.grad(loss, z)
            del loss
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss = f(z, static)
            (g,) = torch.autograd.grad(loss, z)
        for c, (wl, wg) in zip(cases + cases[:1], want + want[:1]):
            with torch.no_grad():
                z.copy_(c.logits)
            for name in ("act_t", "old_t", "adv_t", "ref_t"):
                getattr(static, name).copy_(getattr(c, name))
            torch.randn(100, device=device).sum()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(loss.detach(), wl) and torch.equal(g, wg)


def test_moved_saved_tensors(device, one_pass):
    """Hooks that move what a forward saved (here to the host and back): the backward reads it where
    it is then."""
    off = torch.tensor([0, 5, 9, 16, 22], device=device)
    for vocab in (10, 301, 9001):
        c = Case(24, vocab, torch.bfloat16, device)
        wide = torch.zeros((24, vocab + 5), dtype=torch.bfloat16, device=device)
        wide[:, :vocab] = c.logits
        z = wide[:, :vocab].requires_grad_()
        for f in (lambda: cl.selected_log_probs(z, c.act_t).sum(),
                  lambda: cl.policy_loss(z, c.act_t, c.old_t, c.adv_t) * 0.5,
                  lambda: cl.preference_loss(z, c.act_t, off, c.ref_t)):
            (want,) = torch.autograd.grad(f(), z)
            with torch.autograd.graph.save_on_cpu():
                loss = f()
            junk = [torch.full((1 << 16,), 255, dtype=torch.uint8, device=device) for _ in range(8)]
            (got,) = torch.autograd.grad(loss, z)
            assert torch.equal(got, want)
            del junk
    x = torch.rand(40, 30, device=device, requires_grad=True)
    rng = torch.tensor([3, 4], device=device)
    (want,) = torch.autograd.grad(cl.dropout(x, 0.5, rng).sum(), x)
    with torch.autograd.graph.save_on_cpu():
        y = cl.dropout(x, 0.5, rng).sum()
    assert torch.equal(torch.autograd.grad(y, x)[0], want)


def test_streams(device):
    c = Case(64, 5001, torch.bfloat16, device)
    z = c.logits.requires_grad_()
    ref = cl.policy_loss(z, c.act_t, c.old_t, c.adv_t)
    (gref,) = torch.autograd.grad(ref, z)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        loss = cl.policy_loss(z, c.act_t, c.old_t, c.adv_t)
        (g,) = torch.autograd.grad(loss, z)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(loss, ref) and torch.equal(g, gref)


@pytest.mark.parametrize("rows,vocab,dtype", [
    (20001, 3, torch.float32), (100003, 17, torch.bfloat16), (240000, 60, torch.float32),
    (60000, 220, torch.float32), (60001, 450, torch.bfloat16), (50000, 300, torch.float32),
    (20000, 1300, torch.bfloat16), (4000, 3500, torch.float32), (1700, 8191, torch.float32),
    (900, 16383, torch.float32), (700, 50021, torch.bfloat16), (450, 32767, torch.float32)])
def test_many_rows(device, rows, vocab, dtype):
    """Sizes that take the gradient out of the forward by themselves, and sums over more rows than
    one workgroup adds, against float64 formulas on the device."""
    g = torch.Generator(device=device).manual_seed(rows)
    z = (torch.randn((rows, vocab), generator=g, device=device) * 2.5).to(dtype).requires_grad_()
    a = torch.randint(0, vocab, (rows,), generator=g, device=device)
    a[::7] = IGNORE
    z64 = z.detach().double()
    counted = a != IGNORE
    act = a.clamp(min=0)
    probs = torch.softmax(z64, 1)
    lp = torch.log_softmax(z64, 1).gather(1, act[:, None])[:, 0] * counted
    pick = torch.randint(0, 5, (rows,), generator=g, device=device)
    ratio = torch.tensor([0.4, 0.9, 1.0, 1.15, 1.7], dtype=torch.float64, device=device)
    old = (lp - ratio.log()[pick]).float()
    adv = torch.randn(rows, generator=g, device=device)
    loss, got = cl.policy_loss(z, a, old, adv, return_log_probs=True)
    (grad,) = torch.autograd.grad(loss, z)
    r = torch.exp(lp - old.double())
    A = adv.double()
    term = -torch.minimum(r * A, r.clamp(0.8, 1.2) * A) * counted
    slope = torch.where(r * A <= r.clamp(0.8, 1.2) * A, -r * A, 0.0) * counted / counted.sum()
    err = (vocab / 256 + 40 + float(z64.max() - z64.min())) * 2.0**-24
    assert float((got.double() - lp).abs().max()) <= err + 2.0**-23 * float(lp.abs().max())
    bound = float(A.abs().max()) * 1.8
    assert abs(float(loss.detach()) - float(term.sum() / counted.sum())) <= bound * (err + 2.0**-23)
    ref = -probs * slope[:, None]
    ref.scatter_add_(1, act[:, None], slope[:, None])
    # as Case.check_gradient: errors of the slope and of the probabilities, then one rounding
    far = (2 * err * slope.abs() + 2 * bound * err / float(counted.sum()))[:, None] \
        + ref.abs() * (torch.finfo(dtype).eps / 2 * 1.01) + 1e-37
    assert bool(((grad.double() - ref).abs() <= far).all())
    assert not grad[::7].any()


@pytest.mark.parametrize("pairs,rows", [(1, 9000), (2, 30001), (300, 4000), (5000, 20001)])
def test_preference_of_many_rows(device, pairs, rows):
    """Few long sequences (a workgroup for each pair) and many short ones (a wave for each)."""
    vocab = 6
    c = Case(rows, vocab, torch.float32, device, ignored=0.1)
    rng = np.random.default_rng(pairs)
    cuts = np.sort(rng.integers(0, rows + 1, 2 * pairs - 1))
    offsets = np.concatenate(([0], cuts, [rows - 1]))
    offsets = np.minimum(offsets, rows - 1)
    z = c.logits.requires_grad_()
    loss, h = cl.preference_loss(z, c.act_t, torch.as_tensor(offsets).to(device), c.ref_t,
                                 beta=0.05, return_margins=True)
    want, term, slope = P.preference_terms(c.lp, c.actions, offsets, c.ref, 0.05, 0.0)
    seq = np.diff(offsets)
    herr = 0.05 * (seq[:pairs] + seq[pairs:]) * c.err * 1.01
    _near(_np(h), want, herr, c.wide)
    _near(float(loss.detach()), term.mean(), herr.mean() + np.abs(term).mean() * 2.0**-23, c.wide)
    serr = np.zeros(rows)
    for i in range(pairs):
        e = 0.05 * herr[i] / 4 + 0.1 * 2.0**-24
        serr[offsets[i]:offsets[i + 1]] = e
        serr[offsets[pairs + i]:offsets[pairs + i + 1]] = e
    c.check_gradient(torch.autograd.grad(loss, z)[0], slope / pairs, serr / pairs)


def test_rows_beyond_32_bits(device):
    """Logits whose last rows lie past 2^32 elements, reached through their stride."""
    rows, vocab = 3, 1001
    stride = (1 << 31) + 64
    big = torch.empty(2 * stride + vocab, dtype=torch.float16, device=device)
    x = big.as_strided((rows, vocab), (stride, 1))
    c = Case(rows, vocab, torch.float16, device, ignored=0.0)
    x.copy_(c.logits)
    lp = cl.selected_log_probs(x, c.act_t)
    assert torch.equal(lp, cl.selected_log_probs(c.logits, c.act_t))
    _near(_np(lp), c.lp, c.err, c.wide)


def test_more_than_2_to_32_logits(device):
    """The last rows of 66000 x 65536 logits (8.7 GB), in one pass and in two."""
    rows, vocab = 66000, 65536
    z = torch.empty((rows, vocab), dtype=torch.bfloat16, device=device)
    z.copy_((torch.randn(vocab, device=device) * 2.5).expand(rows, vocab))
    c = Case(4, vocab, torch.bfloat16, device, ignored=0.0)
    z[-4:] = c.logits
    a = torch.full((rows,), IGNORE, device=device)
    a[-4:] = c.act_t
    f = torch.zeros(rows, device=device)
    old, adv = f.clone(), f.clone()
    old[-4:], adv[-4:] = c.old_t, c.adv_t
    z.requires_grad_()
    loss, lp = cl.policy_loss(z, a, old, adv, reduction="sum", return_log_probs=True)
    _near(_np(lp[-4:]), c.lp, c.err, c.wide)
    (g,) = torch.autograd.grad(loss, z)
    term, slope = P.policy_terms(c.lp, c.actions, c.old, c.adv, c.ref, 0.2, 0.2, 0.0)
    c.check_gradient(g[-4:], slope, 4 * np.abs(c.adv) * c.err)
    assert not g[:-4].any()
    del g, loss
    lp = cl.selected_log_probs(z, a)
    (g,) = torch.autograd.grad(lp, z, adv)
    _near(_np(lp[-4:]), c.lp, c.err, c.wide)
    c.check_gradient(g[-4:], c.adv)
    assert not g[:-4].any()


def test_threads_past_32_bits_short_rows(device):
    """2^28 rows and some of two classes, 16 threads each, and half as many pairs."""
    pairs, beta = (1 << 27) + 1, 0.5
    rows = 2 * pairs
    torch.manual_seed(0)
    z = torch.randint(-8, 9, (rows, 2), device=device, dtype=torch.int8).to(torch.bfloat16)
    a = torch.arange(rows, device=device) % 2
    z.requires_grad_()
    loss, h = cl.preference_loss(z, a, torch.arange(rows + 1, device=device), beta=beta,
                                 reduction="sum", return_margins=True)
    (g,) = torch.autograd.grad(loss, z)
    with torch.no_grad():
        d = (z[:, 0].double() - z[:, 1].double()) * (1 - 2 * a)   # chosen less other: -16 .. 16
        lp = torch.nn.functional.logsigmoid(d)
        want = beta * (lp[:pairs] - lp[pairs:])
        err = (2 / 256 + 40 + 16) * 2.0**-24      # of lp (_sum_error)
        assert ((h - want).abs() <= 2 * beta * err + want.abs() * 2.0**-24).all()
        total = float(torch.nn.functional.softplus(-want).sum())
        # per pair beta's two errors and a rounding of the term, 16 at most; the sum's rounding
        assert abs(float(loss) - total) <= pairs * (2 * beta * err + 16 * 2.0**-24) \
            + total * 2.0**-24
        slope = -beta * torch.sigmoid(-want)
        slope = torch.cat((slope, -slope))
        own = slope * torch.sigmoid(-d)
        # 1 - p_a is off by lp's error, the slope by a quarter of the margin's
        off = beta * (err + 2 * beta * err / 4 + 4 * 2.0**-24)
        mine = g.gather(1, a[:, None])[:, 0].double()
        other = g.gather(1, 1 - a[:, None])[:, 0].double()
        assert ((mine - own).abs() <= off + own.abs() * 2.0**-8).all()
        assert ((other + own).abs() <= off + own.abs() * 2.0**-8).all()


def test_threads_past_32_bits_long_rows(device):
    """2^24 rows and some, a workgroup each: the same row of 2050 classes over and over, counted
    at both ends; the gradient (69 GB) in a pass of its own and out of the forward."""
    rows, vocab = (1 << 24) + 3, 2050
    c = Case(6, vocab, torch.bfloat16, device, ignored=0.0, seed=3)
    row = c.logits[0].clone()
    one = np.repeat(_np(row)[None], 6, axis=0)
    lp, probs = P.log_probs(one, c.actions)
    at = torch.tensor([0, 1, 2, rows - 3, rows - 2, rows - 1], device=device)
    a = torch.full((rows,), IGNORE, device=device)
    a[at] = c.act_t
    up = torch.zeros(rows, device=device)
    up[at] = torch.tensor([1.0, -0.5, 2.0, 0.25, -1.0, 3.0], device=device)
    z = row.expand(rows, vocab).requires_grad_()
    err = _sum_error(one, torch.float32)

    def check(got, g):
        _near(_np(got[at]), lp, err, torch.float32)
        slope = _np(up[at])
        own = P.logit_gradient(probs, c.actions, slope)
        # the probabilities' error, both lps' in the ratio, and the exponential's 2^-20
        _near(_np(g[at]), own, np.abs(slope)[:, None] * (3 * err + 2.0**-18), torch.bfloat16)
        assert not got[3:-3].any() and not g[3:-3].any()

    got = cl.selected_log_probs(z, a)
    (g,) = torch.autograd.grad(got, z, up)
    check(got.detach(), g)
    del g
    # ratios of exactly 1 in fp64 are not to be had: inside the range the slope is -A r
    old = torch.zeros(rows, device=device)
    old[at] = got.detach()[at]
    assert policy._prefills(3, rows, vocab)
    loss, got = cl.policy_loss(z, a, old, -up, reduction="sum", return_log_probs=True)
    (g,) = torch.autograd.grad(loss, z)
    check(got, g)
    del g
    torch.cuda.empty_cache()


def test_group_sum_threads_past_32_bits(device):
    """2^24 samples and some, a workgroup each."""
    rows, k = (1 << 24) + 3, 4
    torch.manual_seed(1)
    x = torch.rand((rows, 8), device=device)
    a = torch.arange(rows, device=device) % k
    lp = cl.GroupSum(k, tau=0.25).log_probs(x, a)
    z = x.double().view(rows, k, 2).sum(-1) / 0.25
    want = torch.log_softmax(z, -1).gather(1, a[:, None])[:, 0]
    assert ((lp - want).abs() <= (k / 256 + 40 + 8) * 2.0**-24 + want.abs() * 2.0**-24).all()


def test_no_gradient_is_formed_where_none_is_recorded(device):
    z = torch.randn((8192, 4096), device=device, dtype=torch.bfloat16).requires_grad_()
    a = torch.zeros(8192, dtype=torch.int64, device=device)
    f = torch.zeros(8192, device=device)
    assert policy._prefills(3, 8192, 4096)
    with torch.no_grad():
        want = cl.policy_loss(z, a, f, f + 1)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        got = cl.policy_loss(z, a, f, f + 1)
    assert torch.cuda.max_memory_allocated() - before < z.nbytes // 8
    assert torch.equal(got, want)


def test_calls_are_timed(device):
    """A recorder sees the forward's calls and those of the backward's thread, and their results
    are the untimed ones."""
    z = torch.randn((64, 10), device=device, requires_grad=True)
    a = torch.zeros(64, dtype=torch.int64, device=device)
    x = torch.rand((64, 100), device=device, requires_grad=True)
    off = torch.tensor([0, 30, 64], device=device)
    drop = cl.Dropout(0.5, seed=1).to(device)

    def step():
        lp = cl.selected_log_probs(z, a)
        g = torch.autograd.grad(lp.sum() + cl.policy_loss(z, a, lp.detach(), lp.detach()), z)[0]
        loss = cl.GroupSum(10).preference_loss(x, a, off, reduction="sum")
        return g, torch.autograd.grad(loss, x)[0]

    want = step()
    with timing.record() as rec:
        got = step()
        drop(x)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    names = {"cl_selected_log_prob_forward", "cl_selected_log_prob_backward",
             "cl_policy_loss_forward", "cl_policy_loss_backward", "cl_group_sum_centered_forward",
             "cl_preference_loss_forward", "cl_group_sum_chosen_backward", "cl_dropout_next",
             "cl_dropout"}
    calls = rec.summary()
    assert set(calls) == names and all(v["calls"] == 1 for v in calls.values())
    step()
    assert rec.summary() == calls


def test_threads(device):
    """Two threads, a stream each, call at once."""
    cases = [Case(64, 1000, torch.float32, device, seed=s) for s in (0, 1)]
    torch.cuda.synchronize()

    def step(c):
        z = c.logits.detach().requires_grad_()
        loss = cl.policy_loss(z, c.act_t, c.old_t, c.adv_t, c.ref_t, kl_coef=0.1)
        return torch.cat((loss.detach()[None], torch.autograd.grad(loss, z)[0].flatten()))

    want = [step(c) for c in cases]
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [step(cases[i]) for _ in range(50)]
            torch.cuda.current_stream().synchronize()
        return all(torch.equal(g, want[i]) for g in got)

    with concurrent.futures.ThreadPoolExecutor(2) as ex:
        assert all(ex.map(work, (0, 1)))


def test_checkpointed_and_inference(device):
    """The losses inside of a recomputed segment, and where nothing is recorded."""
    c = Case(48, 1000, torch.float32, device)
    z = c.logits.requires_grad_()
    off = torch.tensor([0, 20, 48], device=device)

    def both(x):
        x = x * 1.0
        return cl.policy_loss(x, c.act_t, c.old_t, c.adv_t, c.ref_t, kl_coef=0.1) \
            + cl.preference_loss(x, c.act_t, off, c.ref_t) \
            + cl.selected_log_probs(x, c.act_t).sum() \
            + cl.dropout(x, 0.5, 7).sum()

    want = both(z)
    (g,) = torch.autograd.grad(want, z)
    for reentrant in (False, True):
        got = torch.utils.checkpoint.checkpoint(both, z, use_reentrant=reentrant)
        assert torch.equal(got, want)
        if reentrant:
            z.grad = None
            got.backward()
            assert torch.equal(z.grad, g)
        else:
            assert torch.equal(torch.autograd.grad(got, z)[0], g)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            got = both(z)
        assert torch.equal(got, want) and not got.requires_grad
    with pytest.raises(RuntimeError):
        torch.func.grad(both)(z.detach())


@pytest.mark.parametrize("layout", ["columns", "rows", "strided"])
@pytest.mark.parametrize("batch,feats,k", [(64, 12000, 10), (1024, 12000, 10), (65, 200001, 10),
                                           (64, 200000, 2), (128, 30000, 300)])
def test_group_sum_methods_sum_in_64_bits(device, batch, feats, k, layout):
    """In every layout a score's error is that of one rounding at the size of its difference from
    the largest one (spread 2^-24), whatever the class sums' size: twice that in lp, which is a
    difference of two such numbers, and the fp64 additions' own, at most gsz + 8 of numbers up to
    gsz.  Class sums in fp32 would be off by some sqrt(gsz) gsz 2^-24 / tau, ten times as much and
    more."""
    rng = np.random.default_rng(feats + k)
    tau, unit, gsz = 2.0, 2.0**-24, -(-feats // k)
    x = torch.as_tensor(rng.random((batch, feats))).float()
    xn = _np(x)
    if layout == "columns":
        x = x.t().contiguous().to(device).t()
    elif layout == "strided":
        x = torch.zeros((batch, 2 * feats), device=device)[:, ::2].copy_(x)
    x = x.to(device).requires_grad_()
    padded = np.zeros((batch, gsz * k))
    padded[:, :feats] = xn
    z = padded.reshape(batch, k, gsz).sum(2) / tau
    # the most likely class, whose log-probability is the smallest number, and any other
    actions = np.where(rng.random(batch) < 0.5, z.argmax(1), rng.integers(0, k, batch))
    lp, probs = P.log_probs(z, actions)
    d = z - z.max(1, keepdims=True)
    err = 2 * -d.min() * unit + 2 * (gsz + 8) * gsz * 2.0**-53 / tau + _sum_error(d, torch.float32)
    got = cl.GroupSum(k, tau).log_probs(x, torch.as_tensor(actions).to(device))
    _near(_np(got), lp, err, torch.float32)
    up = torch.as_tensor(rng.standard_normal(batch)).float().to(device)
    (grad,) = torch.autograd.grad(got, x, up)
    want = P.logit_gradient(probs, actions, _np(up))
    bound = np.abs(_np(up))[:, None] * 2 * err + np.abs(want) * 3 * unit
    spread = np.repeat(np.eye(k), gsz, axis=1)[:, :feats] / tau
    _near(_np(grad), want @ spread, bound @ spread, torch.float32)


@pytest.mark.parametrize("recorded", [False, True])
def test_a_failing_backward_raises_the_package_error(device, recorded):
    """The library refuses a backward whose saved buffer has gone (it checks before any launch);
    its error keeps its type on the way from autograd's thread."""
    c = Case(8, 20, torch.float32, device)
    x = torch.rand((8, 100), device=device, requires_grad=True)
    z = c.logits.requires_grad_()
    off = torch.tensor([0, 3, 8], device=device)
    gs = cl.GroupSum(20)
    calls = [lambda: cl.selected_log_probs(z, c.act_t).sum(),
             lambda: cl.policy_loss(z, c.act_t, c.old_t, c.adv_t),
             lambda: cl.preference_loss(z, c.act_t, off),
             lambda: gs.policy_loss(x, c.act_t, c.old_t, c.adv_t)]

    def lost(t):
        return t[:0].clone() if t.dtype == torch.uint8 else t

    for call in calls:
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lost):
            loss = call()
        with timing.record() if recorded else contextlib.nullcontext():
            with pytest.raises(_capi.CompactLogicError, match=r"cl_.*backward failed.*null"):
                loss.backward()
    assert z.grad is None and x.grad is None
    for call in calls:
        call().backward()
    assert torch.isfinite(z.grad).all() and torch.isfinite(x.grad).all()


@pytest.mark.parametrize("pairs,rows", [(2, 12), (2, 9000), (70, 9000)])
@pytest.mark.parametrize("grouped", [False, True])
def test_rows_inside_a_decrease_of_the_offsets(device, pairs, rows, grouped):
    """Where sequence 1 runs backwards, from row 5 to 3, rows 3 and 4 lie in sequences 0 and 2: no
    order of their kernels' stores decides, the gradient is NaN (0 where the row does not count).
    The other rows of the pairs without a decrease have theirs.  One kernel for few short pairs,
    for long ones, for many."""
    rng = np.random.default_rng(rows + pairs)
    k = 20
    z = rng.standard_normal((rows, k))
    z = torch.as_tensor(z - z.max(1, keepdims=True)).float()      # as GroupSum's scores are centred
    actions = rng.integers(0, k, rows)
    actions[[4, 7]] = IGNORE
    off = np.concatenate(([0, 5, 3], np.linspace(8, rows, 2 * pairs - 2).astype(int)))
    lp, probs = P.log_probs(_np(z), actions)
    h = P.preference_terms(lp, actions, off, None, 0.1, 0.0)[0]
    slope = np.zeros(rows)
    for i in range(pairs):
        d = np.nan if i == 1 else -0.1 / (1 + np.exp(h[i]))
        slope[off[i]:off[i + 1]] = d
        slope[off[pairs + i]:off[pairs + i + 1]] = -d
    slope[3:5] = np.nan
    slope[actions == IGNORE] = 0.0
    x = z.to(device).requires_grad_()               # a class per feature: the scores are x
    act, offsets = torch.as_tensor(actions).to(device), torch.as_tensor(off).to(device)
    loss = cl.GroupSum(k).preference_loss if grouped else cl.preference_loss
    terms = loss(x, act, offsets, reduction="none")
    assert torch.isnan(terms).tolist() == [i == 1 for i in range(pairs)]
    (grad,) = torch.autograd.grad(terms, x, torch.ones_like(terms))
    grad = _np(grad)
    bad = np.isnan(slope)
    assert np.isnan(grad[bad]).all() and (grad[actions == IGNORE] == 0).all()
    # a margin adds gaps of rows of two sequences, each off by the error of its lp
    err = _sum_error(_np(z), torch.float32)
    longest = np.diff(off).max()
    known = np.where(bad, 0.0, slope)
    want = P.logit_gradient(probs, actions, known)
    bound = np.abs(known)[:, None] * 2 * err + 0.1 * (0.1 * 2 * longest * err) \
        + np.abs(want) * 3 * 2.0**-24
    _near(grad[~bad], want[~bad], bound[~bad], torch.float32)
