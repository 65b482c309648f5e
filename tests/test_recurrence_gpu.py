"""The gated recurrence against a walk in float64: every kernel, layout and type, gradients, graphs."""
import numpy as np
import pytest
import torch

import compactlogic_amd as cl
from oracle import recurrence_np as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]
LAYOUTS = ["features", "time_batch", "time_features", "padded", "padded time", "strided", "mixed"]
# one and two steps; one stretch of either length and their borders; several stretches; segments
SHAPES = [(1, 1, 1), (3, 1, 7), (70, 1, 33), (2, 2, 5), (4, 3, 9), (1, 9, 1), (2, 31, 67), (1, 32, 130),
          (3, 33, 5), (2, 64, 3), (2, 128, 2), (5, 129, 1), (1, 255, 12), (2, 256, 65), (2, 257, 8),
          (1, 513, 70), (3, 777, 2), (1, 5003, 3), (2, 2100, 33)]


def _np(t):
    return t.detach().double().cpu().numpy()


def _lay(t, layout):
    """t [batch, time, features] with its values, lying as `layout` says."""
    if layout in ("features", "mixed"):
        return t.contiguous().clone()
    if layout == "time_batch":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "time_features":
        return t.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    b, s, f = t.shape
    if layout == "padded":
        return t.new_zeros((b, s + 1, f + 3))[:, 1:, 1:f + 1].copy_(t)
    if layout == "padded time":
        return t.new_zeros((f, b + 1, s + 5)).permute(1, 2, 0)[1:, 3:s + 3].copy_(t)
    return t.new_zeros((b, 2 * s, 2 * f))[:, ::2, ::2].copy_(t)


def _inputs(shape, dtype, device, seed, mix=True):
    gen = torch.Generator().manual_seed(seed)
    b, s, f = shape
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    g = torch.sigmoid(torch.randn(shape, generator=gen) * 1.5 + 1)
    ends = torch.rand(shape, generator=gen)
    g = torch.where(ends < 0.03, 0.0, torch.where(ends > 0.95, 1.0, g))
    x = torch.rand(shape, generator=gen) if mix else torch.randn(shape, generator=gen)
    return [t.to(dtype).to(device) for t in (x, g, torch.randn(shape, generator=gen))] + \
        [torch.randn((b, f), generator=gen).to(wide).to(device) for _ in range(2)]


def _close(got, want, units, dtype, out=None):
    """`units` roundings of the arithmetic and one of the result's type."""
    out = out or dtype
    u = 2.0**-53 if dtype == torch.float64 else 2.0**-24
    half = torch.finfo(out).eps / 2
    tiny = torch.finfo(out).smallest_normal * torch.finfo(out).eps
    got = _np(got)
    bad = np.abs(got - want) > (units * u + np.abs(want) * half) * 1.001 + tiny
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


def _run_and_check(shape, dtype, device, layout, form, seed):
    x, g, gy, h0, gl = _inputs(shape, dtype, device, seed, form == "mix")
    nx, ng, ngy, nh, ngl = (_np(t) for t in (x, g, gy, h0, gl))
    x, gy = _lay(x, layout), _lay(gy, "strided" if layout == "padded" else layout)
    g = _lay(g, "time_features" if layout == "mixed" else layout)
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    x.requires_grad_(), g.requires_grad_(), h0.requires_grad_()
    y, last = cl.gated_recurrence(x, g, h0, form=form, return_state=True)
    grads = torch.autograd.grad((y, last), (x, g, h0), (gy, gl))
    h, eh = R.forward(nx, ng, nh, form == "mix")
    assert y.shape == x.shape and y.dtype == dtype and last.dtype == wide and last.shape == h0.shape
    _close(y, h, eh, dtype)
    _close(last, h[:, -1], eh[:, -1], dtype, wide)
    for got, (want, err), out in zip(grads, R.backward(nx, ng, nh, ngy, ngl, form == "mix"),
                                     (dtype, dtype, wide)):
        assert got.dtype == out
        _close(got, want, err, dtype, out)
    with torch.no_grad():                     # without a graph: the same bits
        y2, last2 = cl.gated_recurrence(x, g, h0, form=form, return_state=True)
        assert torch.equal(y, y2) and torch.equal(last, last2)
    return x, y, grads


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("form", ["mix", "add"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_matches_a_walk(device, dtype, form, layout):
    for i, shape in enumerate(SHAPES):
        print(shape, flush=True)
        x, y, grads = _run_and_check(shape, dtype, device, layout, form, i)
        if layout == "time_features" and min(shape) > 1:
            for t in (y, *grads[:2]):         # results lie as x does
                assert t.permute(2, 0, 1).is_contiguous()
        if layout in ("features", "strided"):
            assert y.is_contiguous()


# one stretch of 16, up to three of 32, one more step; many workgroups with up to 16 of them, one more step
@pytest.mark.parametrize("shape", [(2, 9, 4), (3, 16, 131), (70, 13, 300), (2, 17, 9), (3, 65, 130), (3, 96, 5),
                                   (3, 97, 5), (512, 17, 6), (513, 48, 5), (512, 49, 6), (512, 100, 6),
                                   (171, 512, 300), (512, 513, 5)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_stretches_of_either_length(device, dtype, shape):
    for layout in ("features", "padded"):
        _run_and_check(shape, dtype, device, layout, "mix" if shape[0] > 3 else "add", 3)


# many sequences: one stretch of 32 lanes, two and three, then 64
@pytest.mark.parametrize("shape", [(41, 65, 50), (2, 128, 1024), (41, 129, 50), (3, 257, 700), (41, 500, 50),
                                   (41, 513, 50), (3, 769, 700)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_lanes_of_either_count(device, dtype, shape):
    for layout in ("time_batch", "padded time"):
        _run_and_check(shape, dtype, device, layout, "add" if shape[0] > 3 else "mix", 4)


@pytest.mark.parametrize("shape", [(300, 1, 1), (1, 1, 300), (300, 40, 1), (1, 40, 300)])
def test_dimensions_of_one(device, shape):
    for layout in LAYOUTS:
        _run_and_check(shape, torch.float32, device, layout, "mix", 7)


def test_gradients_are_differences(device):
    """By float64 differences through the kernels themselves, several stretches and segments."""
    for layout, shape in (("features", (1, 600, 2)), ("time_features", (2, 300, 1)), ("features", (2, 2, 3)),
                          ("time_batch", (2, 6, 3))):
        x, g, _, h0, _ = _inputs(shape, torch.float64, device, 3)
        x, g = _lay(x, layout), _lay(g * 0.9 + 0.05, layout)
        w = torch.randn_like(x)
        for form in ("mix", "add"):
            leaves = [t.detach().requires_grad_() for t in (x, g, h0)]
            def loss(x, g, h0):
                y, last = cl.gated_recurrence(x, g, h0, form=form, return_state=True)
                return (y * w).sum() + (last * last).sum()
            grads = torch.autograd.grad(loss(*leaves), leaves)
            r = np.random.default_rng(0)
            for k, t in enumerate(leaves):
                for _ in range(6):
                    at = tuple(int(r.integers(0, n)) for n in t.shape)
                    with torch.no_grad():
                        d = torch.zeros_like(t)
                        d[at] = 1e-5
                        up, down = ([u + s * d if u is t else u for u in leaves] for s in (1, -1))
                        diff = float(loss(*up) - loss(*down)) / 2e-5
                    assert abs(diff - float(grads[k][at])) < 1e-6 * max(1, abs(diff))


def test_some_gradients_alone(device):
    x, g, gy, h0, gl = _inputs((3, 70, 9), torch.float32, device, 4)
    nx, ng, ngy, nh, ngl = (_np(t) for t in (x, g, gy, h0, gl))
    zero, none = np.zeros_like(ngy), np.zeros_like(nh)
    (dx, ex), (dg, eg), (ds, es) = R.backward(nx, ng, nh, ngy, ngl, True)
    for k, (want, err) in enumerate(((dx, ex), (dg, eg), (ds, es))):
        leaves = [x, g, h0]
        leaves[k] = leaves[k].clone().requires_grad_()
        y, last = cl.gated_recurrence(*leaves, return_state=True)
        (got,) = torch.autograd.grad((y, last), leaves[k], (gy, gl))
        _close(got, want, err, torch.float32)
    for y_grad, l_grad in ((ngy, none), (zero, ngl)):
        a, b, c = (t.clone().requires_grad_() for t in (x, g, h0))
        y, last = cl.gated_recurrence(a, b, c, return_state=True)
        out, up = (y, gy) if y_grad is ngy else (last, gl)
        for got, (want, err) in zip(torch.autograd.grad(out, (a, b, c), up),
                                    R.backward(nx, ng, nh, y_grad, l_grad, True)):
            _close(got, want, err, torch.float32)
    # no state: 0, and its gradient goes nowhere
    a = x.clone().requires_grad_()
    y = cl.gated_recurrence(a, g)
    h, eh = R.forward(nx, ng, none, True)
    _close(y, h, eh, torch.float32)
    (got,) = torch.autograd.grad(y, a, gy)
    (want, err), _, _ = R.backward(nx, ng, none, ngy, none, True)
    _close(got, want, err, torch.float32)


@pytest.mark.parametrize("layout", ["features", "time_features"])
@pytest.mark.parametrize("shape", [(2, 2, 8), (2, 30, 16), (2, 700, 16), (1, 3000, 4)])
def test_ends_of_the_gate_mask(device, shape, layout):
    """0 drops NaN and infinities that came before, 1 leaves NaN inputs unread, in the results and in
    the gradients of x and the state."""
    x, g, gy, h0, gl = _inputs(shape, torch.float32, device, 5)
    cut = shape[1] // 2
    g[:, cut] = 0.0
    x[:, :cut, ::2] = float("nan")
    h0[:, 1::4] = float("inf")
    g[:, cut + 1:, 3] = 1.0                   # holds to the end
    x[:, cut + 1:, 3] = float("nan")
    x, g, gy = (_lay(t, layout).requires_grad_(i < 2) for i, t in enumerate((x, g, gy)))
    y = cl.gated_recurrence(x, g, h0)
    h, eh = R.forward(_np(x), _np(g), _np(h0), True)
    assert torch.isfinite(y[:, cut:]).all() and np.isfinite(h[:, cut:]).all()
    _close(y[:, cut:], h[:, cut:], eh[:, cut:], torch.float32)
    if shape[1] > 2:
        assert torch.isnan(y[:, cut - 1, 0]).all() and not torch.isfinite(y[:, 0, 1]).any()
    (gx,) = torch.autograd.grad(y, x, gy)
    ok = R.backward(_np(x), _np(g), np.where(np.isfinite(_np(h0)), _np(h0), 0), _np(gy), 0 * _np(gl), True)[0]
    _close(gx, *ok, torch.float32)
    # what lies behind a cut does not reach back: gradients that are NaN there
    bad = gy.detach().clone()
    bad[:, cut:] = float("nan")
    (gx,) = torch.autograd.grad(cl.gated_recurrence(x, g, h0), x, bad)
    assert torch.isfinite(gx[:, :cut]).all() and torch.isnan(gx[:, cut]).all()


def test_long_holds_do_not_lose_nan(device):
    """Gates whose product underflows still carry NaN and infinities, as a walk does."""
    x = torch.zeros(1, 2048, 8, device=device)
    g = torch.full_like(x, 0.25)
    x[0, 3, 2] = float("nan")
    for layout in ("features", "time_features"):
        y = cl.gated_recurrence(_lay(x, layout), _lay(g, layout))
        assert torch.isnan(y[0, 3:, 2]).all()
        y[0, :, 2] = 0
        assert (y == 0).all()


def test_exact_on_binary_values(device):
    """A latch: every type and layout, the same bits as the walk."""
    gen = torch.Generator().manual_seed(1)
    for shape in ((3, 300, 17), (2, 7, 5), (4, 1, 9)):
        x, g = ((torch.rand(shape, generator=gen) < 0.5).double() for _ in range(2))
        h0 = (torch.rand((shape[0], shape[2]), generator=gen) < 0.5).double()
        want = R.forward(x.numpy(), g.numpy(), h0.numpy(), True)[0]
        for dtype in DTYPES:
            for layout in LAYOUTS:
                y = cl.gated_recurrence(_lay(x.to(dtype).to(device), layout), _lay(g.to(dtype).to(device), layout),
                                        h0.to(device))
                np.testing.assert_array_equal(_np(y), want)


@pytest.mark.parametrize("layout", ["features", "time_features"])
def test_step_by_step(device, layout):
    """One step at a time from the state handed on, and in two parts, against the whole."""
    x, g, _, h0, _ = _inputs((5, 40, 21), torch.bfloat16, device, 6)
    x, g = _lay(x, layout), _lay(g, layout)
    h, eh = R.forward(_np(x), _np(g), _np(h0), True)
    state = h0
    for t in range(40):
        y, state = cl.gated_recurrence(x[:, t:t + 1], g[:, t:t + 1], state, return_state=True)
        _close(y, h[:, t:t + 1], eh[:, t:t + 1], torch.bfloat16)
        _close(state, h[:, t], eh[:, t], torch.float32)
    y, state = cl.gated_recurrence(x[:, :13], g[:, :13], h0, return_state=True)
    y = cl.gated_recurrence(x[:, 13:], g[:, 13:], state)
    _close(y, h[:, 13:], eh[:, 13:], torch.bfloat16)


def test_broadcast_inputs(device):
    """A gate shared by features or batch entries: its gradient is the sum."""
    x, g, gy, h0, _ = _inputs((4, 50, 12), torch.float32, device, 8)
    for part in (g[:1, :, :1], g[:, :, :1], g[:1]):
        leaf = part.clone().requires_grad_()
        y = cl.gated_recurrence(x, leaf.expand_as(x), h0)
        (got,) = torch.autograd.grad(y, leaf, gy)
        full = _np(part) + np.zeros(x.shape)
        _, (want, err), _ = R.backward(_np(x), full, _np(h0), _np(gy), 0 * _np(h0), True)
        axes = tuple(i for i in range(3) if part.shape[i] == 1 and x.shape[i] > 1)
        n = np.prod([x.shape[i] for i in axes])
        units = err.sum(axes, keepdims=True) + n * np.abs(want).sum(axes, keepdims=True)  # and torch's sum
        _close(got, want.sum(axes, keepdims=True), units, torch.float32)
    state = h0[:1].clone().requires_grad_()
    y = cl.gated_recurrence(x, g, state.expand(4, 12))
    (got,) = torch.autograd.grad(y, state, gy)
    _, _, (want, err) = R.backward(_np(x), _np(g), np.repeat(_np(state), 4, 0), _np(gy), 0 * _np(h0), True)
    _close(got, want.sum(0, keepdims=True), err.sum(0, keepdims=True) + 4 * np.abs(want).sum(0, keepdims=True),
           torch.float32)


def test_empty(device):
    x = torch.zeros(2, 0, 3, device=device, dtype=torch.float16)
    h0 = torch.rand(2, 3, device=device)
    y, last = cl.gated_recurrence(x, x, h0, return_state=True)
    assert y.shape == x.shape and torch.equal(last, h0) and last is not h0
    assert torch.equal(cl.gated_recurrence(x, x, return_state=True)[1], torch.zeros(2, 3, device=device))
    for shape in ((0, 4, 3), (2, 4, 0)):
        x = torch.zeros(shape, device=device).requires_grad_()
        y, last = cl.gated_recurrence(x, x.detach(), return_state=True)
        assert y.shape == shape and last.shape == (shape[0], shape[2])
        y.sum().backward()
        assert x.grad.shape == shape


@pytest.mark.parametrize("layout", ["features", "time_features"])
@pytest.mark.parametrize("shape", [(2, 1, 64), (2, 600, 40)])
def test_graph_replays_like_eager(device, shape, layout):
    x, g, gy, h0, gl = _inputs(shape, torch.float32, device, 9)
    x, g, gy = (_lay(t, layout) for t in (x, g, gy))
    x.requires_grad_(), g.requires_grad_()

    def step():
        y, last = cl.gated_recurrence(x, g, h0, return_state=True)
        return (y, last, *torch.autograd.grad((y, last), (x, g), (gy, gl)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(3):
        with torch.no_grad():
            x.mul_(0.9)
            g.mul_(0.95)
            h0.add_(0.1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b)


def test_another_stream(device):
    x, g, gy, h0, gl = _inputs((2, 1500, 30), torch.float32, device, 10)
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y1 = cl.gated_recurrence(a, g, h0)
        (g1,) = torch.autograd.grad(y1, a, gy)
    s.synchronize()
    y2 = cl.gated_recurrence(b, g, h0)
    (g2,) = torch.autograd.grad(y2, b, gy)
    assert torch.equal(y1, y2) and torch.equal(g1, g2)


def test_refusals(device):
    x = torch.rand(2, 3, 4, device=device)
    for bad in (torch.rand(2, 3, 5, device=device), x.half()):
        with pytest.raises(RuntimeError, match="one shape and dtype"):
            cl.gated_recurrence(x, bad)
    with pytest.raises(RuntimeError, match="one shape"):
        cl.gated_recurrence(x[0], x[0])
    with pytest.raises(RuntimeError, match="dtype"):
        cl.gated_recurrence(x.long(), x.long())
    with pytest.raises(RuntimeError, match="same HIP device"):
        cl.gated_recurrence(x, x.cpu())
    with pytest.raises(ValueError, match="form"):
        cl.gated_recurrence(x, x, form="max")
    with pytest.raises(TypeError, match="state"):
        cl.gated_recurrence(x, x, 0.0)
    for bad in (torch.zeros(2, 3, device=device), torch.zeros(2, 4), torch.zeros(2, 4, device=device).long()):
        with pytest.raises(RuntimeError, match="state"):
            cl.gated_recurrence(x, x, bad)
    y = cl.gated_recurrence(x.requires_grad_(), x)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    # a state of another type is taken over, and gets its gradient in that type
    h0 = torch.rand(2, 4, device=device).bfloat16().requires_grad_()
    (g,) = torch.autograd.grad(cl.gated_recurrence(x, x, h0).sum(), h0)
    assert g.dtype == torch.bfloat16


@pytest.mark.parametrize("layout", ["features", "time_features"])
def test_more_than_32_bits_of_elements(device, layout):
    b, t, f = 2, 70000, 32768                 # 4.6e9 elements of two bytes each
    shape = (b, t, f) if layout == "features" else (f, b, t)
    order = (0, 1, 2) if layout == "features" else (1, 2, 0)
    x = torch.zeros(shape, dtype=torch.bfloat16, device=device).permute(order)
    g = torch.full(shape, 0.5, dtype=torch.bfloat16, device=device).permute(order)
    for i in range(3):
        x[i % b, t - 3 + i, f - 1 - 7 * i] = 1.0 + i
    x.requires_grad_()
    y, last = cl.gated_recurrence(x, g, form="add", return_state=True)
    want = torch.zeros(b, f, device=device)
    for i in range(3):
        want[i % b, f - 1 - 7 * i] = (1.0 + i) * 0.5**(2 - i)
    assert torch.equal(last, want) and torch.equal(y[:, -1].float(), want)
    del y
    up = torch.zeros_like(last)
    up[1, f - 2] = 1.0
    y, last = cl.gated_recurrence(x, g, form="add", return_state=True)
    del y
    (gx,) = torch.autograd.grad(last, x, up)
    got = gx[:, -4:].float()
    want = torch.zeros_like(got)
    want[1, :, f - 2] = torch.tensor([0.125, 0.25, 0.5, 1.0], device=device)
    assert torch.equal(got, want)
    assert float(gx[:, :-200].abs().max()) == 0.0


# ---- the layer

def test_layer_is_its_latches(device):
    """Outputs and all gradients against the two layers' outputs walked in torch, in training."""
    torch.manual_seed(0)
    m = cl.LogicRecurrence(40, 30).to(device)
    x = torch.rand(6, 11, 40, device=device).requires_grad_()
    h0 = torch.rand(6, 30, device=device).requires_grad_()
    y, last = m(x, h0, return_state=True)
    w = torch.randn_like(y)
    grads = torch.autograd.grad((y * w).sum() + last.sum(), [x, h0, m.gate.weights, m.data.weights])
    flat = x.reshape(-1, 40)
    gate, data = (f(flat).double().reshape(6, 11, 30) for f in (m.gate, m.data))
    h, steps = h0.double(), []
    for t in range(11):
        h = gate[:, t] * h + (1 - gate[:, t]) * data[:, t]
        steps.append(h)
    want = torch.stack(steps, 1)
    ref = torch.autograd.grad((want * w).sum() + h.sum(), [x, h0, m.gate.weights, m.data.weights])
    np.testing.assert_allclose(_np(y), _np(want), rtol=2e-6, atol=2e-6)
    for a, b in zip(grads, ref):              # sums of 66 samples' fp32 terms on both sides
        np.testing.assert_allclose(_np(a), _np(b), rtol=1e-4, atol=1e-5)


def test_layer_in_eval_is_a_circuit(device):
    torch.manual_seed(1)
    m = cl.LogicRecurrence(20, 16).to(device).eval()
    x = (torch.rand(3, 50, 20, device=device) < 0.5).float()
    y, last = m(x, return_state=True)
    gate, data = (f(x.reshape(-1, 20)).reshape(3, 50, 16).cpu() for f in (m.gate, m.data))
    h = torch.zeros(3, 16)
    for t in range(50):
        h = torch.where(gate[:, t] == 1, h, data[:, t])
        assert torch.equal(y[:, t].cpu(), h)
    assert torch.equal(last.cpu(), h)
    state, parts = None, []
    for t in range(50):                       # token by token
        part, state = m(x[:, t:t + 1], state, return_state=True)
        parts.append(part)
    assert torch.equal(torch.cat(parts, 1), y)
    m.freeze()
    assert torch.equal(m(x), y)


@pytest.mark.parametrize("shape", [(0, 5), (3, 0)])
def test_layer_without_steps(device, shape):
    m = cl.LogicRecurrence(20, 16).to(device)
    state = torch.rand(shape[0], 16, device=device)
    y, last = m(torch.zeros(*shape, 20, device=device), state, return_state=True)
    assert y.shape == (*shape, 16) and torch.equal(last, state)


def test_layer_in_half(device):
    """float16 sequences through the layers' half path, against its own outputs walked."""
    torch.manual_seed(2)
    m = cl.LogicRecurrence(40, 30).to(device)
    x = torch.rand(4, 16, 40, device=device).half()
    y, last = m(x, return_state=True)
    gate, data = (f(x.reshape(-1, 40)).reshape(4, 16, 30) for f in (m.gate, m.data))
    h, err = R.forward(_np(data), _np(gate), np.zeros((4, 30)), True)
    _close(y, h, err, torch.float16)
    _close(last, h[:, -1], err[:, -1], torch.float16, torch.float32)


def test_gates_outside_of_the_unit_interval(device):
    """Negative and growing gates are as good as any."""
    gen = torch.Generator().manual_seed(3)
    for shape in ((2, 70, 9), (3, 5, 40), (1, 300, 3)):
        x, g = (torch.randn(shape, generator=gen).to(device) for _ in range(2))
        g = (g * 0.4).clamp(-1.3, 1.3)
        for layout in ("features", "time_features"):
            for form in ("mix", "add"):
                a, b = (_lay(t, layout).requires_grad_() for t in (x, g))
                y = cl.gated_recurrence(a, b, form=form)
                zero = np.zeros((shape[0], shape[2]))
                h, err = R.forward(_np(x), _np(g), zero, form == "mix")
                _close(y, h, err, torch.float32)
                gx, gg = torch.autograd.grad(y, (a, b), torch.ones_like(y))
                (wx, ex), (wg, eg), _ = R.backward(_np(x), _np(g), zero, np.ones(shape), zero, form == "mix")
                _close(gx, wx, ex, torch.float32)
                _close(gg, wg, eg, torch.float32)


@pytest.mark.parametrize("layout", ["features", "time_features"])
def test_saved_tensors_may_move(device, layout):
    """Hooks on saved tensors may hand them back with other strides; x and gate may be one tensor."""
    x, g, gy, h0, gl = _inputs((3, 300, 17), torch.float32, device, 11)
    a, b = (_lay(t, layout).requires_grad_() for t in (x, g))
    y = cl.gated_recurrence(a, b, h0)
    want = torch.autograd.grad(y, (a, b), gy)
    for pack in (lambda t: t.cpu(), lambda t: t.contiguous().clone()):
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(device)):
            y = cl.gated_recurrence(a, b, h0)
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, (a, b), gy), want))
    one = cl.gated_recurrence(b, b, h0)
    (got,) = torch.autograd.grad(one, b, gy)
    (wx, ex), (wg, eg), _ = R.backward(_np(g), _np(g), _np(h0), _np(gy), 0 * _np(gl), True)
    _close(got, wx + wg, ex + eg + np.abs(wx) + np.abs(wg), torch.float32)


# A run of steps whose gates multiply past the type's largest number, in every kernel: few steps, one
# stretch and several of either length, narrow rows, segments; 4 to 64 lanes, two stretches, segments.
GROWING = [("features", (2, 8, 12)), ("features", (3, 16, 40)), ("features", (2, 90, 40)),
           ("features", (2, 128, 70)), ("features", (2, 300, 9)), ("features", (512, 100, 6)),
           ("features", (2, 300, 3)), ("features", (1, 3000, 12)), ("features", (1, 3000, 2)),
           ("time_batch", (3, 15, 5)), ("time_features", (3, 31, 7)), ("time_batch", (3, 63, 7)),
           ("time_features", (40, 127, 52)), ("time_batch", (40, 250, 52)), ("time_features", (40, 255, 52)),
           ("time_batch", (3, 500, 4)), ("time_features", (2, 3000, 3))]


def _near(got, want, units, dtype, out=None):
    """_close, and no NaN (which no comparison of magnitudes finds)."""
    assert np.isfinite(want).all() and torch.isfinite(got).all()
    _close(got, want, units, dtype, out)


def _growth(time, dtype, share):
    """A gate whose product over `share` of the time passes the range of the arithmetic; at most what
    the type holds."""
    bits = 1030 if dtype == torch.float64 else 130
    most = {torch.float16: 15.0, torch.float64: 300.0}.get(dtype, 100.0)
    return float(2.0 ** min(most, np.ceil(32 * bits / (share * time)) / 32))


@pytest.mark.parametrize("form", ["mix", "add"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_growing_gates_over_nothing(device, dtype, form):
    """Steps of nothing, however large their gates' product: no state, no inputs up to the last three
    steps, no gradients behind the first three."""
    for layout, shape in GROWING:
        print(layout, shape, flush=True)
        b, s, f = shape
        gate = torch.tensor(_growth(s, dtype, 0.9), dtype=torch.float64).to(dtype)
        x, _, gy, _, gl = _inputs(shape, dtype, device, 12)
        x[:, :-3] = 0
        gy[:, 3:] = 0
        gl.zero_()
        x, gy = (t * 2.0**-10 for t in (x, gy))       # three steps of up to 2^100 each stay in the range
        if float(gate) > 2.0**40:
            x, gy = (t * float(gate)**-1 for t in (x, gy))
        g = torch.full_like(x, float(gate))
        nx, ng, ngy = (_np(t) for t in (x, g, gy))
        none = np.zeros((b, f))
        x, g, gy = (_lay(t, layout) for t in (x, g, gy))
        x.requires_grad_(), g.requires_grad_()
        y, last = cl.gated_recurrence(x, g, form=form, return_state=True)
        h, eh = R.forward(nx, ng, none, form == "mix")
        wide = torch.float64 if dtype == torch.float64 else torch.float32
        if dtype != torch.float16 or np.abs(h).max() < 6e4:
            _near(y, h, eh, dtype)
        _near(last, h[:, -1], eh[:, -1], dtype, wide)
        gx, gg = torch.autograd.grad(y, (x, g), gy)
        (wx, ex), (wg, eg), _ = R.backward(nx, ng, none, ngy, none, form == "mix")
        if dtype != torch.float16 or np.abs(wx).max() < 6e4:
            _near(gx, wx, ex, dtype)
        if dtype != torch.float16 or np.abs(wg).max() < 6e4:
            _near(gg, wg, eg, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
def test_growing_gates_from_a_small_state(device, dtype):
    """A state next to the smallest numbers grows to a large one, and so does a gradient."""
    low, growth = (-1000.0, 1900.0) if dtype == torch.float64 else (-110.0, 200.0)
    for layout, shape in GROWING:
        print(layout, shape, flush=True)
        b, s, f = shape
        gate = float(torch.tensor(2.0 ** (growth / s), dtype=torch.float64).to(dtype))
        if not np.log2(gate) * s + low < (1000 if dtype == torch.float64 else 120):
            continue                                  # (a type of few bits rounds the gate up)
        x, _, gy, h0, gl = _inputs(shape, dtype, device, 13)
        x, gy, h0, gl = (torch.zeros_like(x), torch.zeros_like(gy), h0 * 2.0**low, gl * 2.0**low)
        g = torch.full_like(x, gate)
        nx, ng, ngy, nh, ngl = (_np(t) for t in (x, g, gy, h0, gl))
        x, g, gy = (_lay(t, layout) for t in (x, g, gy))
        x.requires_grad_(), h0.requires_grad_()
        y, last = cl.gated_recurrence(x, g, h0, form="add", return_state=True)
        h, eh = R.forward(nx, ng, nh, False)
        wide = torch.float64 if dtype == torch.float64 else torch.float32
        _near(y, h, eh, dtype)
        _near(last, h[:, -1], eh[:, -1], dtype, wide)
        gx, gs = torch.autograd.grad((y, last), (x, h0), (gy, gl))
        (wx, ex), _, (ws, es) = R.backward(nx, ng, nh, ngy, ngl, False)
        _near(gx, wx, ex, dtype)
        _near(gs, ws, es, dtype, wide)


def test_gates_that_shrink_and_grow(device):
    """Products below the smallest number that grow again, within a thread's steps and beyond them: what
    is left of a large state is what a walk leaves."""
    for layout, shape in GROWING:
        b, s, f = shape
        if s < 8:
            continue
        print(layout, shape, flush=True)
        _, _, _, h0, gl = _inputs(shape, torch.float32, device, 14)
        h0, gl = (t.sign() * 2.0**100 for t in (h0, gl))
        x = torch.zeros(shape, device=device)
        g = torch.ones_like(x)
        g[:, 1:3] = 2.0**-80
        g[:, 3:5] = 2.0**80                           # 2^100, 2^20, 2^-60, 2^20, 2^100
        nx, ng, nh, ngl = (_np(t) for t in (x, g, h0, gl))
        x, g = (_lay(t, layout) for t in (x, g))
        x.requires_grad_()
        y, last = cl.gated_recurrence(x, g, h0, form="add", return_state=True)
        h, _ = R.forward(nx, ng, nh, False)
        assert np.array_equal(_np(y), h) and np.array_equal(_np(last), h[:, -1])
        (gx,) = torch.autograd.grad(last, x, gl)
        with np.errstate(over="ignore"):              # (2^100 times 2^80 is infinite, and stays so)
            c, want = ngl.astype(np.float32), np.empty_like(ng, np.float32)
            for t in range(s - 1, -1, -1):
                want[:, t], c = c, ng[:, t].astype(np.float32) * c
        assert np.array_equal(_np(gx), want)


def test_growth_past_the_range(device):
    """What leaves the range is infinite, and a gate of 0 begins anew."""
    for layout, shape in GROWING:
        if shape[1] < 15:
            continue
        print(layout, shape, flush=True)
        s = shape[1]
        cut = s - s // 4
        x = torch.ones(shape, device=device)
        g = torch.full_like(x, 2.0 ** min(100.0, np.ceil(300 / cut * 8) / 8))
        g[:, cut] = 0.0
        g[:, cut + 1:] = 0.5
        y = cl.gated_recurrence(_lay(x, layout), _lay(g, layout), form="add")
        assert torch.isinf(y[:, cut - 1]).all() and (y[:, cut - 1] > 0).all()
        k = torch.arange(s - cut, device=device, dtype=torch.float64)
        want = (2 - 0.5**k)[None, :, None].expand(shape[0], s - cut, shape[2])
        _near(y[:, cut:], _np(want), 64 * np.ones(want.shape), torch.float32)


@pytest.mark.parametrize("layout", LAYOUTS)
def test_results_are_finite(device, layout):
    """NaN passes a comparison of magnitudes: none where inputs are finite."""
    for i, shape in enumerate(SHAPES):
        for dtype in (torch.float32, torch.bfloat16):
            for t in _run_and_check(shape, dtype, device, layout, "mix", i)[1:]:
                assert all(torch.isfinite(v).all() for v in (t if isinstance(t, tuple) else (t,)))


def test_forward_mode_is_refused(device):
    """Tangents are not dropped without a word, whichever argument has them."""
    import torch.autograd.forward_ad as fw
    x, g, _, h0, _ = _inputs((2, 6, 5), torch.float32, device, 15)
    for k in range(3):
        args = [x, g, h0]
        with fw.dual_level():
            args[k] = fw.make_dual(args[k], torch.ones_like(args[k]))
            for on in (True, False):
                with torch.set_grad_enabled(on), pytest.raises(RuntimeError, match="jvp"):
                    cl.gated_recurrence(*args)
