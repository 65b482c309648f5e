"""verify_drafts without a device: refusals, the C entry point's checks, the oracle's distribution."""
import ctypes

import numpy as np
import pytest
import torch

import compactlogic_amd as cl
from compactlogic_amd import _capi
from oracle import verify_np as V


def test_refusals_without_a_device():
    z, t, u = torch.zeros(2, 3, 4), torch.zeros(2, 2, dtype=torch.int64), torch.zeros(2, 3)
    with pytest.raises(RuntimeError, match="HIP device"):
        cl.verify_drafts(z, t, None, u)
    for args in ((None, t, None, u), (z, [1], None, u), (z, t, None, 0.5)):
        with pytest.raises(TypeError):
            cl.verify_drafts(*args)


def test_c_arguments_are_checked_before_the_device():
    lib = _capi.load()
    bad, ok = _capi.CL_ERR_INVALID_ARGUMENT, _capi.CL_OK
    need = ctypes.c_int64()

    def size(dtype=0, s=2, k=3, v=10):
        return lib.cl_verify_drafts_workspace(dtype, s, k, v, ctypes.byref(need))

    assert size() == ok and need.value == 0
    assert size(v=4096) == ok and need.value == 0
    assert size(v=8193) == ok and need.value >= 2 * 7 * 2 * 8 + 2 * 32 + 2 * 5 * 24
    assert size(dtype=4) == bad and size(s=-1) == bad and size(k=-1) == bad and size(v=0) == bad
    assert size(s=1 << 30, v=8193) == bad and b"too many" in lib.cl_last_error()
    assert size(v=1 << 60) == bad and size(k=1 << 60) == bad and size(s=1 << 60) == bad
    assert lib.cl_verify_drafts_workspace(0, 1, 1, 1, None) == bad

    def rc(dtype=0, z=8, zs=(40, 10), q=8, qs=(30, 10), t=8, u=8, ud=0, s=2, k=3, v=10, out=8, acc=8, lp=8,
           ws=None, wb=0):
        return lib.cl_verify_drafts(dtype, z, *zs, q, *qs, t, -100, u, ud, s, k, v, out, acc, lp, ws, wb, None)

    assert rc(s=0) == ok
    for name in ("z", "t", "u", "out", "acc", "lp"):
        assert rc(**{name: None}) == bad, name
    assert rc(dtype=9) == bad and rc(ud=2) == bad and rc(zs=(-1, 10)) == bad and rc(qs=(30, -10)) == bad
    assert rc(v=9000) == bad and b"workspace" in lib.cl_last_error()
    assert rc(v=9000, ws=8, wb=1 << 20) == bad
    assert rc(s=0) == ok and lib.cl_last_error() == b""


def test_oracle_draws_as_the_target():
    """Whatever the draft: of n draws the share of each token lies within 5 standard deviations."""
    r = np.random.default_rng(0)
    n = 20000
    p, q = np.array([0.5, 0.2, 0.3, 0.0]), np.array([0.1, 0.6, 0.2, 0.1])
    with np.errstate(divide="ignore"):
        z, d = np.log(p), np.log(q)
    drafts = r.choice(4, (n, 1), p=q)
    out, accepted, lp = V.verify(np.broadcast_to(z, (n, 2, 4)), drafts, np.broadcast_to(d, (n, 1, 4)), r.random((n, 2)))
    share = np.bincount(out[:, 0], minlength=4) / n
    assert np.all(np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / n))
    assert abs(accepted.mean() - np.minimum(p, q).sum()) < 5 * 0.5 / np.sqrt(n)
    second = out[accepted == 1, 1]
    share = np.bincount(second, minlength=4) / len(second)
    assert np.all(np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / len(second)))
    np.testing.assert_allclose(lp[:, 0], np.log(p[out[:, 0]]))
