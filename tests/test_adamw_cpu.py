"""FusedAdamW without a device: its refusals, the C entry points' checks, the oracle of 8-bit moments."""
import copy
import ctypes
import pickle
import warnings

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


def test_rounding_is_checked_and_warned_of():
    p = torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(ValueError, match="rounding"):
        cl.FusedAdamW([p], rounding="up")
    for betas, bits, rounding, warned in (((0.9, 0.999), 8, "nearest", True), ((0.95, 0.9), 8, "nearest", True),
                                          ((0.9, 0.9), 8, "nearest", False), ((0.9, 0.999), 8, "random", False),
                                          ((0.9, 0.999), 32, "nearest", False)):
        with warnings.catch_warnings(record=True) as seen:
            warnings.simplefilter("always")
            opt = cl.FusedAdamW([torch.nn.Parameter(torch.zeros(1))], betas=betas, state_bits=bits, rounding=rounding)
        assert [("betas above 0.9" in str(w.message)) for w in seen] == [True] * warned
        assert opt.param_groups[0]["rounding"] == rounding
    other = cl.FusedAdamW([p], state_bits=8, rounding="random")
    other.load_state_dict(cl.FusedAdamW([p], lr=0.5).state_dict())
    assert other.param_groups[0]["rounding"] == "random" and other.param_groups[0]["lr"] == 0.5


def _run_held(betas, gradient, steps, n, at_random):
    """Moments held in 8 bits over `steps`, the same in float64, and the sizes of the last updates."""
    m = v = np.zeros(n)
    fm, fv = np.zeros(n), np.zeros(n)
    for t in range(1, steps + 1):
        g = gradient(t)
        m1, v1 = A.step32(g, m, v, 1.0, betas)
        fm, fv = betas[0] * fm + (1 - betas[0]) * g, betas[1] * fv + (1 - betas[1]) * g.astype(np.float64)**2
        m, v = A.values(*A.hold(m1, v1, A.words(t, n) if at_random else None))
    sizes = [np.mean(np.abs(a) / (np.sqrt(b) + 1e-12)) for a, b in ((m1, v1), (fm, fv))]
    return m, v, fm, fv, sizes[0] / sizes[1]


def _trajectories():
    r = np.random.default_rng(3)
    n = 2048
    flat = (np.where(r.random(n) < 0.5, -1, 1) * r.uniform(0.5, 2, n)).astype(np.float32)
    noise = r.standard_normal((64, n)).astype(np.float32)
    at = lambda t: np.roll(noise[t % 64], t)
    return n, {"flat": ((0.9, 0.999), lambda t: flat, 2500), "noise": ((0.9, 0.999), at, 2500),
               "shrinks": ((0.9, 0.98), lambda t: at(t) * np.float32(1 if t < 400 else 0.1), 1200)}


@pytest.mark.parametrize("name", ["flat", "noise", "shrinks"])
def test_rounded_at_random_moments_follow(name):
    """Thousands of steps.  A held value's rounding has mean 0 and a variance of at most (what the step
    changes) x (the codes' distance, 1/8 of v): for v at most (1 - b2)(g^2 + v) v / 8, which sums up with
    weights b2^2k to v^2 / 8 at most (E g^2 = v), for |m| at most m E|g| / 8 + m^2 / 8 likewise, below a
    fourth of the mean g^2.  A mean over 2048 elements is within 6 deviations, 6 sqrt(1/4 / 2048) = 0.07.
    The root's mean is off by 3/8 of v's relative variance more, 0.05."""
    n, runs = _trajectories()
    betas, gradient, steps = runs[name]
    m, v, fm, fv, sizes = _run_held(betas, gradient, steps, n, True)
    assert abs(v.mean() / fv.mean() - 1) < 0.07
    scale = np.sqrt(fv.mean())
    assert abs(np.mean((m - fm) * np.sign(fm)) / scale) < 0.07
    assert abs(sizes - 1) < 0.12


def test_rounded_to_the_nearest_moments_stay():
    """What the warning is about: exp_avg_sq next to its first steps' values, or those before gradients
    shrank.  With betas of 0.9 it follows: it moves where (1 - b2) |g^2 - v| is above v / 16 (rising, codes
    up to 1/8 apart) or v / 18 (falling, 1/9), which leaves g^2 / 1.625 to g^2 / (1 - 10/18)."""
    n, runs = _trajectories()
    betas, gradient, steps = runs["flat"]
    _, v, _, fv, sizes = _run_held(betas, gradient, steps, n, False)
    assert v.mean() < 0.1 * fv.mean() and sizes > 3
    betas, gradient, steps = runs["shrinks"]
    _, v, _, fv, sizes = _run_held(betas, gradient, steps, n, False)
    assert v.mean() > 50 * fv.mean() and sizes < 0.2
    for name in ("flat", "shrinks"):
        _, gradient, steps = runs[name]
        _, v, _, fv, _ = _run_held((0.9, 0.9), gradient, steps, n, False)
        assert 1 / 1.625 < v.mean() / fv.mean() < 2.25


def test_random_words_and_codes():
    """Uniform words, and codes that are one of a value's two neighbours, up as often as their distance
    says, itself where it is one; NaN, 0 and the smallest as by the nearest."""
    w = A.words(7, 1 << 16, 3)
    halves = np.concatenate([w & 0xFFFF, w >> np.uint32(16)]) / 65536.0
    assert abs(halves.mean() - 0.5) < 6 * np.sqrt(1 / 12 / len(halves))
    assert abs(np.corrcoef(w & 0xFFFF, w >> np.uint32(16))[0, 1]) < 6 / np.sqrt(len(w))
    assert not np.array_equal(w, A.words(8, 1 << 16, 3)) and np.array_equal(w[2048:], A.words(7, (1 << 16) - 2048, 4))
    n = 1 << 14
    m, v = np.full(n, 1.03, np.float32), np.full(n, 1.03, np.float32)
    m[::256] = v[::256] = 1.0                # (a code itself: 128 and 1 with their blocks' powers)
    got_m, got_v = A.values(*A.hold(m, v, A.words(1, n)))
    for got in (got_m, got_v):
        assert np.all(got[::256] == 1.0)
        rest = np.delete(got, np.arange(0, n, 256))
        assert set(np.unique(rest)) == {1.0, 1.125}
        p = 0.03 / 0.125
        assert abs(np.mean(rest == 1.125) - p) < 6 * np.sqrt(p * (1 - p) / len(rest))
    small = np.full(512, 2.0**-12, np.float32)      # held as 2^-5 and 1/8 of it apart
    small[0] = 1.0
    small[1:256] += np.float32(2.0**-18)
    cm, _, powers = A.hold(small, small, A.words(2, 512))
    got = A.values(cm, np.zeros(512, np.uint8), powers)[0]
    assert set(np.unique(got[1:256])) == {2.0**-12, 2.0**-12 + 2.0**-15} and np.all(got[256:] == 2.0**-12)
    small[1:256] = np.float32(2.0**-15 + 2.0**-18)  # below the normal codes of m, where they are 2^-16 apart
    cm, _, powers = A.hold(small, small, A.words(2, 512))
    got = A.values(cm, np.zeros(512, np.uint8), powers)[0]
    assert set(np.unique(got[1:256])) == {2.0**-15, 2.0**-15 + 2.0**-16}
    odd = np.zeros(256, np.float32)
    odd[:4] = np.nan, 0.0, 1e-30, 1.0
    cm, cv, _ = A.hold(odd, odd, A.words(3, 256))
    assert (cm[0] & 127, cv[0], cm[1], cv[1], cv[2]) == (127, 255, 0, 0, 1)


def test_copies_keep_their_settings():
    p = torch.nn.Parameter(torch.zeros(4))
    opt = cl.FusedAdamW([p], max_norm=3.0, state_bits=8)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert other.max_norm == 3.0 and other.param_groups[0]["state_bits"] == 8


def test_pickles_without_a_rounding_go_on():
    p = torch.nn.Parameter(torch.zeros(4))
    opt = cl.FusedAdamW([p])
    del opt.param_groups[0]["rounding"], opt.defaults["rounding"]
    old = pickle.loads(pickle.dumps(opt))
    assert old.param_groups[0]["rounding"] == "nearest"
    old.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2))]})
    old.load_state_dict(old.state_dict())
    assert [g["rounding"] for g in old.param_groups] == ["nearest"] * 2


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


def test_unknown_rounding_is_refused_by_the_library():
    lib = _capi.load()
    t = _capi.AdamWTensor(16, 16, 16, 16, 16, 10, 0, 8, 0, 2)
    g = _capi.AdamWGroup(1e-3, 0.9, 0.999, 1e-8, 0.0)
    assert lib.cl_adamw_step(1, ctypes.addressof(t), 1, ctypes.addressof(g), 0.0, 8, 8, 1 << 20, None) \
        == _capi.CL_ERR_INVALID_ARGUMENT and b"rounding" in lib.cl_last_error()
    assert lib.cl_adamw_moments_read(0, None, None) == _capi.CL_OK and lib.cl_last_error() == b""


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
