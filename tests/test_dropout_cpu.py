"""The dropout oracle against published vectors, and what dropout refuses without a device."""
import numpy as np
import pytest
import torch
import torch.utils.checkpoint

import compactlogic_amd as cl
from compactlogic_amd import _capi, dropout_layer
from oracle import dropout_np as D


@pytest.mark.parametrize("counter,key,words", [
    # the known answers of philox4x32-10 published with the generator
    ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
     (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1)),
])
def test_oracle_generator_known_answers(counter, key, words):
    got = D.philox(np.array(counter, dtype=np.uint64), np.array(key, dtype=np.uint64))
    assert tuple(int(w) for w in got) == words


def test_oracle_mask_rate():
    """Of n independent bits of rate q, the share lies within 5 standard deviations."""
    keep = D.keep_mask(500, 1003, 0.3, 12345, 7)
    q, n = 1 - D.threshold(0.3) / 65536, keep.size
    assert abs(keep.mean() - q) < 5 * np.sqrt(q * (1 - q) / n)


def test_refusals_without_a_device():
    x = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="HIP device"):
        cl.dropout(x, 0.5, 1)
    with pytest.raises(TypeError):
        cl.dropout([1.0], 0.5, 1)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            cl.Dropout(p)
    with pytest.raises(ValueError, match="64 bits"):
        cl.Dropout(0.5, seed=2**63)


def test_module_without_a_device():
    torch.manual_seed(0)
    a, b = cl.Dropout(0.3), cl.Dropout(0.3)
    assert int(a.rng[0]) != int(b.rng[0])            # every module its own sequence
    torch.manual_seed(0)
    assert torch.equal(cl.Dropout(0.3).rng, a.rng)   # reproducible from torch's seed
    x = torch.rand(3, 5)
    assert a.eval()(x) is x and cl.Dropout(0.0)(x) is x
    assert set(a.state_dict()) == {"rng"} and "p=0.3" in repr(a)


def test_c_arguments_are_checked_before_the_device():
    lib = _capi.load()

    def rc(x=1, xs=(8, 1), y=1, ys=(8, 1), rows=4, cols=8, t=5, dtype=0):
        return lib.cl_dropout(dtype, x, *xs, y, *ys, rows, cols, t, 1, 0.0, 0, 0, None, None)

    bad = _capi.CL_ERR_INVALID_ARGUMENT
    assert rc(rows=0) == _capi.CL_OK
    assert rc(t=65537) == bad and rc(t=0) == bad and rc(t=-1) == bad
    assert rc(rows=-1) == bad and rc(rows=2**32) == bad and rc(cols=2**32) == bad
    assert rc(x=None) == bad and rc(y=None) == bad
    assert rc(dtype=9) == bad and b"dtype" in lib.cl_last_error()
    assert rc(xs=(1, 4)) == bad and b"same dimension" in lib.cl_last_error()
    assert rc(xs=(16, 2), ys=(16, 2)) == bad
    assert rc(xs=(-8, 1)) == bad
    assert rc(ys=(7, 1)) == bad and b"overlap" in lib.cl_last_error()
    assert rc(rows=2**31, cols=2**31, xs=(2**31, 1), ys=(2**31, 1)) == bad
    assert lib.cl_dropout_next(None, None, None) == bad
    assert rc(rows=0) == _capi.CL_OK and lib.cl_last_error() == b""


@pytest.fixture
def plain_dropout(monkeypatch):
    """The module on CPU tensors: the oracle's masks, and the count of calls kept on the CPU."""
    def next_mask(rng):
        used = rng.clone()
        rng[1] += 1
        return used

    def dropout(x, p, rng, fill=None):
        keep = torch.as_tensor(D.keep_mask(*x.shape, p, *(int(v) for v in rng)))
        return torch.where(keep, x, 0.0)

    native = type("Native", (), {"dropout_next": staticmethod(next_mask)})
    monkeypatch.setattr(dropout_layer._native, "load", lambda: native)
    monkeypatch.setattr(dropout_layer._dl, "_check", lambda t, name: None)
    monkeypatch.setattr(dropout_layer, "dropout", dropout)
    return dropout


@pytest.mark.parametrize("reentrant", [False, True])
def test_module_refuses_to_draw_again_in_a_backward(plain_dropout, reentrant):
    """A recomputed segment would drop other elements than the loss saw.  With the mask taken
    before the segment the gradient is that of the mask."""
    x = torch.rand(20, 30, generator=torch.Generator().manual_seed(0)).requires_grad_()
    drop = cl.Dropout(0.5, seed=3)
    y = torch.utils.checkpoint.checkpoint(lambda h: drop(h * h).sum(), x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="next_rng"):
        y.backward()
    assert int(drop.rng[1]) == 1

    rng = drop.next_rng()
    y = torch.utils.checkpoint.checkpoint(lambda h: plain_dropout(h * h, drop.p, rng).sum(), x,
                                          use_reentrant=reentrant)
    y.backward()
    keep = torch.as_tensor(D.keep_mask(20, 30, 0.5, 3, 1))
    assert torch.equal(x.grad, torch.where(keep, 2 * x.detach(), 0.0))
    assert int(drop.rng[1]) == 2
    drop.eval()                                      # the identity may be run again
    x.grad = None
    torch.utils.checkpoint.checkpoint(lambda h: drop(h * h).sum(), x,
                                      use_reentrant=reentrant).backward()
    assert torch.equal(x.grad, 2 * x.detach())
