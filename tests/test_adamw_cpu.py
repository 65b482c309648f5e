"""FusedAdamW without a device: its refusals, the C entry points' checks, the oracle of 8-bit moments."""
import copy
import ctypes
import pickle

import numpy as np
import pytest
import torch

import compactlogic_amd as cl
from compactlogic_amd import _capi
from oracle import adamw_np as A


def test_hyper_parameters_are_checked():
    p = torch.nn.Parameter(torch.zeros(4))
    for bad in (dict(lr=-1.0), dict(eps=-1e-9), dict(weight_decay=-0.1), dict(betas=(1.0, 0.9)),
                dict(betas=(0.9, -0.1)), dict(lr=float("nan")), dict(state_bits=16)):
        with pytest.raises(ValueError):
            cl.FusedAdamW([p], **bad)
        with pytest.raises(ValueError):
            cl.FusedAdamW([torch.nn.Parameter(torch.zeros(1))]).add_param_group(
                {"params": [p], **bad})
    with pytest.raises(ValueError, match="twice"):
        cl.FusedAdamW([p, p])


def test_host_parameters_are_refused():
    p = torch.nn.Parameter(torch.zeros(4))
    opt = cl.FusedAdamW([p])
    opt.step()                                # nothing to do
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="HIP"):
        opt.step()
    with pytest.raises(RuntimeError, match="moments"):
        opt.moments([p])
    assert opt.moments() == ([], [])


def test_state_dicts_of_other_algorithms_are_refused():
    p = torch.nn.Parameter(torch.zeros(4))
    other = torch.optim.AdamW([p], amsgrad=True)
    with pytest.raises(RuntimeError, match="amsgrad"):
        cl.FusedAdamW([p]).load_state_dict(other.state_dict())


def test_groups_without_a_decay_keep_theirs():
    """FusedAdam's groups have none; those of other algorithms lack more."""
    p, q = torch.nn.Parameter(torch.zeros(4)), torch.nn.Parameter(torch.zeros(3))
    other = cl.FusedAdam([{"params": [p]}, {"params": [q]}], lr=0.25, betas=(0.5, 0.75), eps=1e-4)
    opt = cl.FusedAdamW([{"params": [p], "weight_decay": 0.5}, {"params": [q], "state_bits": 8}], weight_decay=0.125)
    opt.load_state_dict(other.state_dict())
    for group, decay, bits in zip(opt.param_groups, (0.5, 0.125), (32, 8)):
        assert set(group) >= {"params", "lr", "betas", "eps", "weight_decay", "state_bits"}
        assert (group["lr"], tuple(group["betas"]), group["eps"]) == (0.25, (0.5, 0.75), 1e-4)
        assert group["weight_decay"] == decay and group["state_bits"] == bits
    assert opt.param_groups[0]["params"][0] is p
    with pytest.raises(RuntimeError, match="betas"):
        opt.load_state_dict(torch.optim.SGD([{"params": [p]}, {"params": [q]}], lr=0.1).state_dict())


def test_fused_adam_refuses_moments_in_8_bits():
    """Their codes would be taken for values."""
    p = torch.nn.Parameter(torch.zeros(4))
    held = cl.FusedAdamW([p], state_bits=8).state_dict()
    held["state"] = {0: {"exp_avg": torch.zeros(4, dtype=torch.uint8).view(torch.float8_e4m3fn),
                         "exp_avg_sq": torch.full((4,), 200, dtype=torch.uint8),
                         "exponents": torch.ones(2, dtype=torch.uint8), "step": torch.tensor(1.0)}}
    opt = cl.FusedAdam([p])
    with pytest.raises(RuntimeError, match="8 bits"):
        opt.load_state_dict(held)
    assert not opt.state


def test_copies_keep_their_settings():
    p = torch.nn.Parameter(torch.zeros(4))
    opt = cl.FusedAdamW([p], max_norm=3.0, state_bits=8)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert other.max_norm == 3.0 and other.param_groups[0]["state_bits"] == 8


def test_c_arguments_are_checked_before_the_device():
    lib = _capi.load()
    bad = _capi.CL_ERR_INVALID_ARGUMENT

    def rc(tensors=(), groups=((1e-3, 0.9, 0.999, 1e-8, 0.0),), step=8, ws=8, ws_bytes=1 << 20):
        ts = (_capi.AdamWTensor * max(1, len(tensors)))(*[_capi.AdamWTensor(*t) for t in tensors])
        gs = (_capi.AdamWGroup * max(1, len(groups)))(*[_capi.AdamWGroup(*g) for g in groups])
        return lib.cl_adamw_step(len(tensors), ctypes.addressof(ts), len(groups),
                                 ctypes.addressof(gs), 0.0, step, ws, ws_bytes, None)

    good = (16, 16, 16, 16, None, 10, 0, 32, 0, 0)
    swap = lambda **k: tuple(k.get(f, v) for (f, _), v in zip(_capi.AdamWTensor._fields_, good))
    for t in (swap(param=None), swap(grad=None), swap(exp_avg=None), swap(exp_avg_sq=None),
              swap(bits=8), swap(bits=4), swap(dtype=9), swap(dtype=-1), swap(numel=-1),
              swap(numel=1 << 50), swap(group=1), swap(group=-1), swap(dtype=1, bits=8, powers=16)):
        assert rc([t]) == bad and lib.cl_last_error() != b"", t
    assert rc([good], step=None) == bad and rc([good], ws=None) == bad
    assert rc([good], ws_bytes=100) == bad and b"workspace" in lib.cl_last_error()
    assert rc([good], ws=12) == bad
    for g in ((-1.0, 0.9, 0.9, 0, 0), (1, 1.0, 0.9, 0, 0), (1, 0.9, float("nan"), 0, 0),
              (1, 0.9, 0.9, -1, 0), (1, 0.9, 0.9, 0, -1)):
        assert rc([good], groups=(g,)) == bad
    assert rc([good], groups=((1, 0.9, 0.9, 0, 0),) * 33) == bad and b"32" in lib.cl_last_error()
    assert lib.cl_adamw_workspace(3, None) == bad and lib.cl_adamw_workspace(-1, None) == bad
    for name in ("cl_adamw_moments_read", "cl_adamw_moments_write"):
        t = _capi.AdamWTensor(*good)
        assert getattr(lib, name)(1, ctypes.addressof(t), None) == bad   # 32 bits
        assert getattr(lib, name)(-1, None, None) == bad and getattr(lib, name)(1, None, None) == bad
        assert getattr(lib, name)(0, None, None) == _capi.CL_OK


def test_oracle_holds_its_own_values():
    """Every code's value is held as that code, and rounding stays within half a step."""
    e = np.append(A._e4m3(), -A._e4m3())
    k = np.zeros(256)
    k[:254], k[254:] = e, 128.0        # the largest of the block in [128, 256)
    k[np.abs(k) >= 256] = 0
    v = np.zeros(256)
    v[:254] = A._e5m3()[1:]
    v[v >= 2] = 0
    cm, cv, powers = A.hold(k, v)
    m2, v2 = A.values(cm, cv, powers)
    np.testing.assert_array_equal(m2, k)
    np.testing.assert_array_equal(v2, v)
    r = np.random.default_rng(0)
    m, v = r.standard_normal(1000).astype(np.float32), r.random(1000).astype(np.float32)
    m2, v2 = A.values(*A.hold(m, v))
    top = np.repeat(np.abs(np.append(m, np.zeros(24))).reshape(-1, 256).max(1), 256)[:1000]
    assert np.all(np.abs(m2 - m) <= np.maximum(np.abs(m) * 2.0**-4, top * 2.0**-17))
    assert np.all(np.abs(v2 - v) <= np.maximum(v * 2.0**-4, 2.0**-31))
    # against torch's own e4m3
    t = torch.tensor(m)
    own = torch.ldexp(t, torch.tensor(3)).to(torch.float8_e4m3fn)
    ours = A._e4m3()[A._nearest(np.abs(m.astype(np.float64)) * 8, A._e4m3())]
    np.testing.assert_array_equal(own.float().abs().numpy(), ours)
