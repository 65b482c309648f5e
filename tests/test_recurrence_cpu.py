"""The gated recurrence without a device: refusals, the C entry points' checks, the oracle."""
import ctypes

import numpy as np
import pytest
import torch

import compactlogic_amd as cl
from compactlogic_amd import _capi
from oracle import recurrence_np as R


def test_refusals_without_a_device():
    x = torch.zeros(2, 3, 4)
    with pytest.raises(TypeError):
        cl.gated_recurrence(x, 0.5)
    with pytest.raises(RuntimeError, match="HIP device"):
        cl.gated_recurrence(x, x)
    with pytest.raises(RuntimeError, match="packed"):
        cl.LogicRecurrence(4, 4)(cl.PackBitsTensor.from_packed(torch.zeros(4, 1, dtype=torch.int64)))
    with pytest.raises(RuntimeError, match="batch, time, 4"):
        cl.LogicRecurrence(4, 4)(torch.zeros(3, 4))


def test_module_holds_two_layers():
    m = cl.LogicRecurrence(6, 5, connections="original", num_gates=8)
    assert m.gate.num_gates == 8 and m.data.connections == "original" and "6, 5" in repr(m)
    m.freeze()
    assert m.gate.is_frozen and m.data.is_frozen


def test_c_arguments_are_checked_before_the_device():
    lib = _capi.load()
    bad, ok = _capi.CL_ERR_INVALID_ARGUMENT, _capi.CL_OK
    S = ctypes.c_int64 * 3
    a, b = ctypes.c_int64(), ctypes.c_int64()
    keep = []

    def addr(s):
        keep.append(S(*s, *(0,) * (3 - len(s))))
        return ctypes.addressof(keep[-1])

    def size(dtype=0, order=0, batch=2, time=3, features=4):
        return lib.cl_recurrence_sizes(dtype, order, batch, time, features, ctypes.byref(a), ctypes.byref(b))

    assert size() == ok and (a.value, b.value) == (0, 0)
    assert size(time=1000) == ok and a.value == 8 * 8 and b.value > 0     # 8 stretches of 128 steps
    assert size(order=9) == bad and size(dtype=7) == bad and size(batch=-1) == bad
    assert size(order=3) == bad and b"one step" in lib.cl_last_error()
    assert size(order=3, time=1) == ok
    assert lib.cl_recurrence_sizes(0, 0, 1, 1, 1, None, None) == bad

    def fwd(dtype=0, order=0, form=0, x=8, xs=(12, 4, 1), g=8, gs=(12, 4, 1), h=None, hs=(4, 1), dims=(2, 3, 4),
            y=8, ys=(12, 4, 1), last=8, ls=(4, 1), ws=None, wb=0):
        return lib.cl_recurrence_forward(dtype, order, form, x, addr(xs), g, addr(gs), h, addr(hs), *dims, y,
                                         addr(ys), last, addr(ls), None, ws, wb, None)

    assert fwd(dims=(0, 3, 4)) == ok and fwd(dims=(2, 3, 0)) == ok
    assert fwd(dims=(2, 0, 4)) == bad and b"no steps" in lib.cl_last_error()
    assert fwd(form=2) == bad and fwd(x=None) == bad and fwd(g=None) == bad and fwd(y=None) == bad
    assert fwd(last=None) == bad and fwd(dtype=5) == bad
    assert fwd(xs=(12, 4, 2)) == bad and b"contiguous" in lib.cl_last_error()
    assert fwd(gs=(-12, 4, 1)) == bad and fwd(ys=(12, 1, 3)) == bad
    assert fwd(order=1) == bad and fwd(order=2) == bad and fwd(h=8, hs=(-4, 1)) == bad
    assert fwd(dims=(2, 1000, 4)) == bad and b"workspace" in lib.cl_last_error()

    def bwd(starts=None, dims=(2, 3, 4), form=0, x=8, ws=None, wb=0):
        s = addr((dims[1] * 4, 4, 1))
        return lib.cl_recurrence_backward(0, 0, form, x, s, 8, s, None, None, starts, None, None, None, None,
                                          *dims, None, None, None, None, None, None, ws, wb, None)

    assert bwd(form=5) == bad and bwd(x=None) == bad and bwd(dims=(2, 0, 4)) == bad
    assert bwd(dims=(2, 1000, 4)) == bad and b"starts" in lib.cl_last_error()
    assert bwd(dims=(2, 1000, 4), starts=8) == bad and b"workspace" in lib.cl_last_error()
    assert bwd(dims=(0, 3, 4)) == ok


@pytest.mark.parametrize("mix", [True, False])
def test_oracle_gradients_are_differences(mix):
    r = np.random.default_rng(0)
    x, g, gy = r.random((3, 2, 9, 4))
    h0, gl = r.random((2, 2, 4))
    loss = lambda x, g, h0: np.sum(R.forward(x, g, h0, mix)[0] * gy) + np.sum(R.forward(x, g, h0, mix)[0][:, -1] * gl)
    grads = [v for v, _ in R.backward(x, g, h0, gy, gl, mix)]
    for k, a in enumerate((x, g, h0)):
        for _ in range(20):
            at = tuple(r.integers(0, n) for n in a.shape)
            d = np.zeros_like(a)
            d[at] = 1e-6
            args = [x, g, h0]
            up, down = list(args), list(args)
            up[k], down[k] = a + d, a - d
            assert abs((loss(*up) - loss(*down)) / 2e-6 - grads[k][at]) < 1e-7
