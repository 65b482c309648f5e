"""What the losses on chosen log-probabilities refuse without a device, and their oracle against
differences."""
import ctypes
import sys
import types

import numpy as np
import pytest
import torch

import compactlogic_amd as cl
from compactlogic_amd import _capi, _native
from oracle import policy_np as P


def test_refusals_without_a_device():
    z, a, f = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64), torch.zeros(3)
    off = torch.tensor([0, 1, 2])
    for call in (lambda: cl.selected_log_probs(z, a), lambda: cl.policy_loss(z, a, f, f),
                 lambda: cl.preference_loss(z, a, off),
                 lambda: cl.GroupSum(5).log_probs(z, a)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()
    with pytest.raises(TypeError):
        cl.selected_log_probs([1.0], a)


def test_c_arguments_are_checked_before_the_device():
    lib = _capi.load()
    ok, bad = _capi.CL_OK, _capi.CL_ERR_INVALID_ARGUMENT

    def lp(dtype=0, x=1, stride=8, rows=2, cols=8, act=1, out=1, state=1):
        return lib.cl_selected_log_prob_forward(dtype, x, stride, rows, cols, act, -100, out, state,
                                                None, 0, None)

    def policy(low=0.2, kl=0.0, ref=None, red=2, loss=1, old=1, rows=2, grad=None):
        return lib.cl_policy_loss_forward(0, 1, 8, rows, 8, 1, -100, old, 1, ref, low, 0.2, kl, red,
                                          1, 1, 1, loss, loss, grad, None, 0, None)

    def pref(pairs=1, smooth=0.0, off=1, red=2, gaps=1):
        return lib.cl_preference_loss_forward(0, 1, 8, 2, 8, 1, -100, None, off, pairs, 0.1, smooth,
                                              red, 1, 1, gaps, 1, 1, 1, 1, 1, 1, None, 0, None)

    assert lp(rows=0, x=None, act=None, out=None, state=None) == ok
    assert lp(cols=0) == bad and lp(cols=2**31) == bad and lp(rows=-1) == bad
    assert lp(rows=2**31) == bad and lp(stride=-1) == bad and lp(dtype=7) == bad
    assert lp(x=None) == bad and lp(act=None) == bad and lp(out=None) == bad
    assert lp(state=None) == bad
    # few long rows are split over workgroups that meet in a workspace
    need = ctypes.c_int64()
    assert lib.cl_token_loss_workspace(0, 4, 1 << 17, ctypes.byref(need)) == ok and need.value > 0
    assert lp(rows=4, cols=1 << 17, stride=1 << 17) == bad and b"workspace" in lib.cl_last_error()
    assert lib.cl_token_loss_workspace(0, 4, 10, ctypes.byref(need)) == ok and need.value == 0
    assert lib.cl_token_loss_workspace(0, 4, 0, ctypes.byref(need)) == bad
    # more classes than one workgroup holds are not summed for a loss
    assert lib.cl_group_sum_centered_workspace_size(0, 64, 900, 1, 512, ctypes.byref(need)) == ok
    assert need.value >= 512 * 64 * 4
    assert lib.cl_group_sum_centered_workspace_size(0, 64, 900, 1, 513, ctypes.byref(need)) == ok
    assert need.value == -1
    assert lib.cl_group_sum_centered_forward(0, 1, 64, 900, 1, 64, 513, 1.0, 1, 1, 1, None) == bad
    assert lib.cl_group_sum_centered_forward(0, 1, 64, 900, 1, 64, 10, 1.0, 1, None, 0, None) == bad
    def chosen(batch=4, k=10, scores=1, up=1, sb=1, pairs=0, seq=None, slope=None):
        return lib.cl_group_sum_chosen_backward(0, scores, batch, 100, k, 1.0, 1, 1, up, None, None,
                                                seq, slope, None, pairs, 1, sb, 4, None)

    assert chosen(batch=0) == ok
    assert chosen(batch=-1) == bad and chosen(k=0) == bad and chosen(scores=None) == bad
    assert chosen(up=None) == bad and b"upstream" in lib.cl_last_error()
    assert chosen(sb=-1) == bad and chosen(pairs=-1) == bad and chosen(pairs=2, seq=1) == bad
    assert policy(low=-0.1) == bad and policy(low=float("nan")) == bad
    assert policy(kl=0.1) == bad and b"KL" in lib.cl_last_error()
    assert policy(red=3) == bad and policy(loss=None) == bad and policy(old=None) == bad
    assert policy(red=0, loss=None, grad=1) == bad and b"scalar" in lib.cl_last_error()
    assert pref(pairs=-1) == bad and pref(smooth=1.5) == bad and pref(off=None) == bad
    assert pref(red=-1) == bad and pref(gaps=None) == bad
    assert lib.cl_selected_log_prob_backward(0, 1, 8, 2, 8, 1, 1, None, 1, None) == bad
    assert lib.cl_policy_loss_backward(0, 1, 8, 2, 8, 1, 1, 2, 1, None, 0, 1, None) == bad
    assert lib.cl_policy_loss_backward(0, 1, 8, 2, 8, 1, 1, 0, 1, None, 1, 1, None) == bad
    assert lib.cl_policy_loss_backward(2, 1, 8, 2, 8, 1, 1, 2, 1, 1, 1, 1, None) == bad
    assert b"type" in lib.cl_last_error()
    yes = ctypes.c_int()
    for dtype, rows, cols, want in [(0, 8192, 4096, 1), (3, 8192, 4096, 1), (2, 8192, 4096, 0),
                                    (1, 8192, 4096, 0), (0, 128, 10, 0), (3, 4096, 65536, 1),
                                    (3, 4096, 65537, 0), (0, 4096, 32768, 1), (0, 4096, 32769, 0)]:
        assert lib.cl_policy_loss_prefills(dtype, rows, cols, ctypes.byref(yes)) == ok
        assert yes.value == want, (dtype, rows, cols)
    assert lib.cl_preference_loss_backward(0, 1, 8, 2, 8, 1, 1, None, 1, 1, 2, 1, 1, 1, None) == bad
    assert lp(rows=0) == ok and lib.cl_last_error() == b""


def _difference(f, z, eps=1e-6):
    g = np.zeros(z.shape)
    for i in np.ndindex(*z.shape):
        hi, lo = z.copy(), z.copy()
        hi[i] += eps
        lo[i] -= eps
        g[i] = (f(hi) - f(lo)) / (2 * eps)
    return g


def test_oracle_gradients_against_differences():
    """Central differences at 1e-6: truncation about 1e-12, cancellation about 1e-16 / 1e-6."""
    rng = np.random.default_rng(0)
    z, actions = rng.standard_normal((6, 5)), np.array([0, 4, -100, 2, 1, 3])
    lp, probs = P.log_probs(z, actions)
    # ratios well inside and outside the clipped range
    old = lp - np.log([0.5, 0.95, 1.0, 1.1, 1.6, 1.05])
    adv, ref = rng.standard_normal(6), lp + 0.3 * rng.standard_normal(6)

    def policy(zz):
        return P.policy_terms(P.log_probs(zz, actions)[0], actions, old, adv, ref, 0.2, 0.28,
                              0.05)[0].sum()

    slope = P.policy_terms(lp, actions, old, adv, ref, 0.2, 0.28, 0.05)[1]
    np.testing.assert_allclose(P.logit_gradient(probs, actions, slope), _difference(policy, z),
                               atol=1e-8)
    offsets = [0, 2, 4, 5, 6]

    def preference(zz):
        return P.preference_terms(P.log_probs(zz, actions)[0], actions, offsets, ref, 0.7,
                                  0.1)[1].sum()

    slope = P.preference_terms(lp, actions, offsets, ref, 0.7, 0.1)[2]
    np.testing.assert_allclose(P.logit_gradient(probs, actions, slope), _difference(preference, z),
                               atol=1e-8)


def test_autograd_extension(monkeypatch):
    """Built, and refused where it is missing or of another torch."""
    built = _native.load()
    assert {"selected_log_probs", "policy_loss", "preference_loss", "dropout",
            "dropout_next"} <= set(dir(built))
    assert _native.load() is built
    monkeypatch.setattr(_native, "_module", None)
    monkeypatch.delattr(cl, "_autograd")
    monkeypatch.setitem(sys.modules, "compactlogic_amd._autograd", None)
    with pytest.raises(_capi.CompactLogicError, match="compactlogic_amd.build"):
        _native.load()
    other = types.SimpleNamespace(torch_version="0.0.1")
    monkeypatch.setattr(cl, "_autograd", other, raising=False)
    monkeypatch.setitem(sys.modules, "compactlogic_amd._autograd", other)
    with pytest.raises(_capi.CompactLogicError, match="torch 0.0.1"):
        _native.load()


def test_a_failing_call_raises_the_package_error():
    """Sizes are refused before anything is allocated or launched."""
    with pytest.raises(_capi.CompactLogicError, match="cl_token_loss_workspace failed.*bad shape"):
        _native.load().selected_log_probs(torch.zeros(3, 0), torch.zeros(3, dtype=torch.int64),
                                          -100, 0, 1.0)
