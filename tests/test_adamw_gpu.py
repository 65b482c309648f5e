"""FusedAdamW against the same step in float64, moments in 8 bits code by code."""
import copy
import io

import numpy as np
import pytest
import torch

import compactlogic_amd as cl
from oracle import adamw_np as A

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]
SHAPES = [(1,), (7,), (3, 5), (255,), (256,), (257,), (2048,), (2049,), (4096 + 13,), (100, 41), (), (0,)]


def _np(t):
    return t.detach().double().cpu().numpy()


def _params(shapes, dtype, device, seed=0, offset=0):
    """Parameters with gradients, `offset` elements off their storage's start."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for s in shapes:
        n = int(np.prod(s))
        make = lambda k: (torch.randn(n + offset, generator=g) * k).to(dtype).to(device)[offset:].view(s)
        p = torch.nn.Parameter(make(1.0))
        p.grad = make(0.1)
        out.append(p)
    return out


def _check(got, want, err, dtype):
    """Within the float32 error, and a storage rounding of 16-bit parameters; float64 arithmetic has
    2^-53 in the place of 2^-24."""
    if dtype == torch.float64:
        err = err * 2.0**-29
    half = 0 if dtype in (torch.float32, torch.float64) else torch.finfo(dtype).eps / 2
    tiny = 2.0**-25 if dtype == torch.float16 else 2.0**-134 if dtype == torch.bfloat16 else 2.0**-150
    assert np.all(np.abs(got - want) <= err + np.abs(want) * half * 1.001 + tiny), \
        float(np.max(np.abs(got - want)))


@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("max_norm", [None, 0.5])
@pytest.mark.parametrize("dtype", DTYPES)
def test_step_in_32_bits(device, dtype, max_norm, offset):
    params = _params(SHAPES, dtype, device, offset=offset)
    groups = [{"params": params[::2], "weight_decay": 0.3, "lr": 0.02},
              {"params": params[1::2], "weight_decay": 0.0, "betas": (0.5, 0.8), "eps": 1e-3}]
    opt = cl.FusedAdamW(groups, lr=0.01, max_norm=max_norm)
    held = {}
    for t in range(1, 4):
        scale = A.scale_of([_np(p.grad) for p in params], max_norm)
        assert max_norm is None or scale < 1
        before = [_np(p) for p in params]
        opt.step()
        for group in opt.param_groups:
            for p in group["params"]:
                i = next(j for j, q in enumerate(params) if q is p)
                m, v = held.get(i, (np.zeros(p.shape), np.zeros(p.shape)))
                (wp, ep), (wm, em), (wv, ev) = A.step(before[i], _np(p.grad), m, v, t, scale, group["lr"],
                                                      group["betas"], group["eps"], group["weight_decay"])
                st = opt.state[p]
                wide = torch.float64 if dtype == torch.float64 else torch.float32
                assert st["exp_avg"].dtype == wide and float(st["step"]) == t
                _check(_np(p), wp, ep, dtype)
                _check(_np(st["exp_avg"]), wm, em, wide)
                _check(_np(st["exp_avg_sq"]), wv, ev, wide)
                held[i] = _np(st["exp_avg"]), _np(st["exp_avg_sq"])
        for p in params:
            p.grad = -0.7 * p.grad


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("max_norm", [None, 0.5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_step_in_8_bits(device, dtype, max_norm, offset):
    """Parameters as with the moments before they are rounded, codes equal."""
    params = _params(SHAPES, dtype, device, offset=offset)
    with torch.no_grad():
        params[8].grad[300:600] *= 1e-6          # a block of small numbers
        params[9].grad[:20] = 0                  # and zeros
    betas, lr, eps, decay = (0.9, 0.98), 0.01, 1e-8, 0.1
    opt = cl.FusedAdamW(params, lr=lr, betas=betas, eps=eps, weight_decay=decay, max_norm=max_norm,
                        state_bits=8)
    held = [(np.zeros(p.shape), np.zeros(p.shape)) for p in params]
    for t in range(1, 5):
        scale = A.scale_of([_np(p.grad) for p in params], max_norm)
        before = [_np(p) for p in params]
        opt.step()
        first, second = opt.moments(params)
        for i, p in enumerate(params):
            g, (m, v) = _np(p.grad), held[i]
            (wp, ep), _, _ = A.step(before[i], g, m, v, t, scale, lr, betas, eps, decay)
            _check(_np(p), wp, ep, dtype)
            cm, cv, powers = A.hold(*A.step32(g, m, v, scale, betas))
            st = opt.state[p]
            np.testing.assert_array_equal(st["exp_avg"].view(torch.uint8).cpu().numpy().reshape(-1), cm)
            np.testing.assert_array_equal(st["exp_avg_sq"].cpu().numpy().reshape(-1), cv)
            np.testing.assert_array_equal(st["exponents"].cpu().numpy(), powers)
            m, v = A.values(cm, cv, powers)
            held[i] = m.reshape(p.shape), v.reshape(p.shape)
            assert first[i].dtype == torch.bfloat16
            np.testing.assert_array_equal(_np(first[i]), held[i][0])
            np.testing.assert_array_equal(_np(second[i]), held[i][1])
        for p in params:
            p.grad = (p.grad * (-0.7 if t % 2 else 3.0)).to(dtype)


def test_extremes_in_8_bits(device):
    """Infinities and NaN stay in their own elements; the smallest and largest numbers keep within
    their format."""
    p = torch.nn.Parameter(torch.zeros(1024, device=device))
    r = np.random.default_rng(1)
    g = r.standard_normal(1024).astype(np.float32)
    g[5], g[9], g[300] = np.inf, np.nan, -np.inf
    g[512:768] = 2.0**-149
    g[768:] = 1e19
    g[800] = 1e-19
    p.grad = torch.tensor(g, device=device)
    betas = (0.9, 0.99)
    opt = cl.FusedAdamW([p], betas=betas, max_norm=None, weight_decay=0.0, state_bits=8)
    opt.step()
    with np.errstate(over="ignore", invalid="ignore"):
        cm, cv, powers = A.hold(*A.step32(g, np.zeros(1024), np.zeros(1024), 1.0, betas))
    st = opt.state[p]
    got = st["exp_avg"].view(torch.uint8).cpu().numpy()
    nan = np.array([5, 9, 300])
    assert np.all((got[nan] & 0x7F) == 0x7F)
    keep = np.setdiff1d(np.arange(1024), nan)
    np.testing.assert_array_equal(got[keep], cm[keep])
    np.testing.assert_array_equal(st["exp_avg_sq"].cpu().numpy(), cv)
    np.testing.assert_array_equal(st["exponents"].cpu().numpy(), powers)
    assert torch.isnan(p[[5, 9, 300]]).all() and torch.isfinite(p[torch.tensor(keep, device=device)]).all()
    first, second = (t[0] for t in opt.moments([p]))
    np.testing.assert_array_equal(_np(first)[keep], A.values(cm, cv, powers)[0][keep])
    assert torch.isnan(first[nan]).all() and torch.isnan(second[nan]).all()


def test_many_tensors_of_every_type(device):
    """More tensors than a launch takes, types and bits mixed: each as if it were alone."""
    r = np.random.default_rng(2)
    sizes = [int(n) for n in r.integers(1, 6000, 150)]
    params = [p for i, n in enumerate(sizes)
              for p in _params([(n,)], DTYPES[i % 4], device, seed=i)]
    small = [p for i, p in enumerate(params) if i % 4 != 1 and i % 3 == 0]
    rest = [p for p in params if all(p is not q for q in small)]
    alone = [copy.deepcopy(p) for p in params]
    opt = cl.FusedAdamW([{"params": rest}, {"params": small, "state_bits": 8}], max_norm=None)
    for p, q in zip(params, alone):
        q.grad = p.grad.clone()
        bits = 8 if any(p is s for s in small) else 32
        one = cl.FusedAdamW([q], max_norm=None, state_bits=bits)
        one.step()
        one.step()
    opt.step()
    opt.step()
    assert all(torch.equal(p, q) for p, q in zip(params, alone))
    # one norm over all of them
    norm = np.sqrt(sum(float(np.sum(_np(p.grad)**2)) for p in params))
    a, b = [copy.deepcopy(p) for p in params], [copy.deepcopy(p) for p in params]
    for p, q, s in zip(params, a, b):
        q.grad = p.grad.clone()
        s.grad = p.grad.clone()
    c = 2.0**-3
    oa = cl.FusedAdamW(a, max_norm=norm * c)
    ob = cl.FusedAdamW(b, max_norm=None, eps=1e-8 / c)
    oa.step()
    ob.step()
    for p, q in zip(oa.moments()[0], ob.moments()[0]):
        np.testing.assert_allclose(_np(p), _np(q) * c, rtol=1e-5, atol=0)


@pytest.mark.parametrize("bits", [32, 8])
def test_hundreds_of_tensors_captured(device, bits):
    """Several launches of one type, whose addresses a graph keeps; and one launch more or less."""
    for count in (16, 17, 128, 129, 300):
        shapes = [((7 * i) % 613 + 1,) for i in range(count)]
        ps, qs = (_params(shapes, torch.float32, device, seed=count) for _ in range(2))
        op, oq = (cl.FusedAdamW(x, max_norm=0.2, state_bits=bits) for x in (ps, qs))
        op.step()
        oq.step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            oq.step()
        for _ in range(3):
            for p, q in zip(ps, qs):
                p.grad.mul_(-0.9)
                q.grad.copy_(p.grad)
            op.step()
            graph.replay()
            torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs))
        scale = A.scale_of([_np(p.grad) for p in ps], 0.2)
        before, (m, v) = [_np(p) for p in ps], ([_np(t) for t in ts] for ts in op.moments())
        op.step()
        for i, p in enumerate(ps):
            (want, err), _, _ = A.step(before[i], _np(p.grad), m[i], v[i], 5, scale, 1e-3, (0.9, 0.999), 1e-8, 0.01)
            _check(_np(p), want, err, torch.float32)


def test_gradients_lie_anywhere_and_may_be_missing(device):
    p, q = _params([(64, 33), (50,)], torch.float32, device)
    g = p.grad.clone()
    p2 = torch.nn.Parameter(p.detach().clone())
    p.grad = g.t().contiguous().t()
    assert not p.grad.is_contiguous()
    p2.grad = g.clone()
    q.grad = None
    before = q.detach().clone()
    opt, opt2 = cl.FusedAdamW([p, q]), cl.FusedAdamW([p2])
    opt.step()
    opt2.step()
    assert torch.equal(p, p2) and torch.equal(q, before) and q not in opt.state
    assert torch.equal(p.grad, g)                       # left as they were
    q.grad = torch.ones_like(q)                         # later, under the shared count
    opt.step()
    assert float(opt.state[q]["step"]) == 2


def test_state_dicts_interchange(device):
    """With torch.optim.AdamW's, between 32 and 8 bits, through a file."""
    def fresh():
        return _params([(300, 7), (513,)], torch.bfloat16, device, seed=5)

    a = fresh()
    opt = cl.FusedAdamW(a, max_norm=None)
    for _ in range(3):
        opt.step()
    file = io.BytesIO()
    torch.save(opt.state_dict(), file)
    file.seek(0)
    b = [copy.deepcopy(p) for p in a]
    for p, q in zip(a, b):
        q.grad = p.grad.clone()
    again = cl.FusedAdamW(b, max_norm=None)
    again.load_state_dict(torch.load(file, weights_only=True))
    assert again.state[b[0]]["exp_avg"].dtype == torch.float32   # not the parameters' type
    again.step()
    opt.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and float(again.state[b[1]]["step"]) == 4

    f = [torch.nn.Parameter(p.detach().float()) for p in fresh()]
    other = torch.optim.AdamW(f, lr=0.01)
    for p in f:
        p.grad = torch.randn_like(p)
    other.step()
    g = [copy.deepcopy(p) for p in f]
    own = cl.FusedAdamW(g, max_norm=None)
    own.load_state_dict(copy.deepcopy(other.state_dict()))       # (the tensors are shared else)
    for p, q in zip(f, g):
        p.grad = torch.randn_like(p)
        q.grad = p.grad.clone()
    other.step()
    own.step()
    for p, q in zip(f, g):
        np.testing.assert_allclose(_np(q), _np(p), rtol=1e-6, atol=1e-8)
    torch.optim.AdamW(f).load_state_dict(own.state_dict())

    small = cl.FusedAdamW([copy.deepcopy(p) for p in g], max_norm=None, state_bits=8)
    small.load_state_dict(own.state_dict())
    ps = small.param_groups[0]["params"]
    for p, q in zip(ps, g):
        cm, cv, powers = A.hold(own.state[q]["exp_avg"].cpu().numpy(), own.state[q]["exp_avg_sq"].cpu().numpy())
        st = small.state[p]
        np.testing.assert_array_equal(st["exp_avg"].view(torch.uint8).cpu().numpy().reshape(-1), cm)
        np.testing.assert_array_equal(st["exp_avg_sq"].cpu().numpy().reshape(-1), cv)
        np.testing.assert_array_equal(st["exponents"].cpu().numpy(), powers)
    file = io.BytesIO()
    torch.save(small.state_dict(), file)
    file.seek(0)
    same = cl.FusedAdamW([copy.deepcopy(p) for p in ps], max_norm=None, state_bits=8)
    same.load_state_dict(torch.load(file, weights_only=True))
    back = cl.FusedAdamW([copy.deepcopy(p) for p in ps], max_norm=None)
    back.load_state_dict(small.state_dict())
    for o in (same, back):
        for x, y in zip(o.moments(), small.moments()):
            assert all(torch.equal(s.float(), t.float()) for s, t in zip(x, y))
    assert "exponents" not in back.state[back.param_groups[0]["params"][0]]


def test_copied_optimizer_goes_on(device):
    (p,) = _params([(700,)], torch.float32, device)
    opt = cl.FusedAdamW([p], state_bits=8)
    opt.step()
    q, o = copy.deepcopy((p, opt))
    q.grad = p.grad.clone()
    assert o.param_groups[0]["params"][0] is q
    opt.step()
    o.step()
    assert torch.equal(p, q) and float(o.state[q]["step"]) == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_graph_replays_like_eager_steps(device, bits):
    eager, graphed = (_params([(5000,), (33, 9)], torch.bfloat16, device) for _ in range(2))
    oe, og = (cl.FusedAdamW(ps, lr=0.01, max_norm=0.3, state_bits=bits) for ps in (eager, graphed))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        oe.step()
        og.step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        og.step()
    for k in range(4):
        for p, q in zip(eager, graphed):
            p.grad.mul_(-1.5)
            q.grad.copy_(p.grad)
        oe.step()
        g.replay()
        torch.cuda.synchronize()
        for p, q in zip(eager, graphed):
            assert torch.equal(p, q)
        for x, y in zip(oe.moments(), og.moments()):
            assert all(torch.equal(s, t) for s, t in zip(x, y))
        assert float(og.state[graphed[0]]["step"]) == 2 + k


def test_first_step_is_refused_in_a_capture(device, monkeypatch):
    (p,) = _params([(10,)], torch.float32, device)
    opt = cl.FusedAdamW([p])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="capture"):
        opt.step()
    monkeypatch.undo()
    opt.step()
    (q,) = _params([(10,)], torch.float32, device)
    opt.add_param_group({"params": [q]})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="capture"):
        opt.step()
    assert float(opt.state[p]["step"]) == 1


def test_changed_settings_between_steps(device):
    """Bits, hyper-parameters and the gradients' types as they are at each call."""
    p, q = _params([(300,), (40,)], torch.float32, device)
    opt = cl.FusedAdamW([{"params": [p]}, {"params": [q]}], max_norm=None)
    opt.step()
    m = opt.state[p]["exp_avg"].clone()
    opt.param_groups[0]["state_bits"] = 8
    opt.param_groups[0]["lr"] = opt.param_groups[0]["weight_decay"] = 0.0
    before = p.detach().clone()
    opt.step()
    assert torch.equal(p, before) and "exponents" in opt.state[p]
    cm, _, powers = A.hold(m.cpu().numpy(), np.zeros(300))
    held = A.values(cm, np.zeros(300, np.uint8), powers)[0]
    want, _ = A.step32(_np(p.grad), held, np.zeros(300), 1.0, (0.9, 0.999))
    cm, _, powers = A.hold(want, np.zeros(300))
    np.testing.assert_array_equal(_np(opt.moments([p])[0][0]), A.values(cm, np.zeros(300, np.uint8), powers)[0])
    first, second = opt.moments()
    assert first[0].dtype == torch.bfloat16 and first[1].dtype == torch.float32
    p.grad, p.grad_dtype = None, torch.float64
    p.grad = torch.ones(300, dtype=torch.float64, device=device)
    with pytest.raises(RuntimeError, match="dtype"):
        opt.step()


def test_another_stream_and_reproducible(device):
    runs = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        ps = _params([(300_001,), (77,)], torch.float32, device, seed=9)
        opt = cl.FusedAdamW(ps, max_norm=0.1)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            opt.step()
            opt.step()
        torch.cuda.synchronize()
        runs.append([p.detach().clone() for p in ps])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_norms_that_are_not_finite(device):
    (p,) = _params([(100,)], torch.float32, device)
    p.grad[3] = float("inf")
    before = p.detach().clone()
    cl.FusedAdamW([p], max_norm=1.0, weight_decay=0.0).step()     # scale 0: inf * 0 in its own place
    assert torch.isnan(p[3])
    keep = torch.arange(100, device=device) != 3
    assert torch.equal(p[keep], before[keep])


def test_autograd_sees_the_step(device):
    (p,) = _params([(10,)], torch.float32, device)
    y = (p * p).sum()
    cl.FusedAdamW([p]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals(device):
    (p,) = _params([(8, 4)], torch.float64, device)
    with pytest.raises(RuntimeError, match="float64"):
        cl.FusedAdamW([p], state_bits=8).step()
    q = torch.nn.Parameter(torch.zeros(8, 4, device=device).t())
    q.grad = torch.zeros_like(q)
    with pytest.raises(RuntimeError, match="contiguous"):
        cl.FusedAdamW([q]).step()
    w = torch.nn.Parameter(torch.zeros(6, 3, device=device))
    w.grad = torch.zeros(6, 3, device=device).to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        cl.FusedAdamW([w]).step()
    c = torch.nn.Parameter(torch.zeros(4, device=device, dtype=torch.complex64))
    c.grad = torch.zeros_like(c)
    with pytest.raises(RuntimeError, match="dtype"):
        cl.FusedAdamW([c]).step()
    a = torch.nn.Parameter(torch.zeros(4, device=device))
    a.grad = torch.ones_like(a)
    opt = cl.FusedAdamW([a])
    opt.step()
    opt.state[a]["exp_avg"] = torch.zeros(5, device=device)
    with pytest.raises(RuntimeError, match="shape"):
        opt.step()


def test_trains_a_network(device):
    """The framework's own layers and loss, a captured step among eager ones."""
    torch.manual_seed(0)
    model = torch.nn.Sequential(cl.LogicLayer(64, 96), cl.LogicLayer(96, 80), cl.GroupSum(10, 2.0)).to(device)
    x = (torch.rand(48, 64, device=device) < 0.4).float()
    y = torch.randint(0, 10, (48,), device=device)
    opt = cl.FusedAdamW(model.parameters(), lr=0.02, state_bits=8)
    ref = [p.detach().clone() for p in model.parameters()]
    for _ in range(3):
        opt.zero_grad(set_to_none=True)
        model[-1].cross_entropy(model[:-1](x), y).backward()
        opt.step()
    assert all(torch.isfinite(p).all() and not torch.equal(p, q)
               for p, q in zip(model.parameters(), ref))


@pytest.mark.parametrize("numel", [3, 2048, 5000])
@pytest.mark.parametrize("bits", [32, 8])
def test_roots_of_the_smallest_moments(device, bits, numel):
    """An exp_avg_sq below the smallest normal number has a root, also where eps is 0 or next to it."""
    for eps in (0.0, 1e-21):
        (p,) = _params([(numel,)], torch.float32, device)
        # the square of a gradient, times 1 - beta2, from 2^-148 to 2^-120
        e = torch.arange(numel, device=device) % 57
        p.grad = torch.exp2(-72.5 + e / 4) * torch.where(e % 2 == 0, 1.0, -1.0)
        opt = cl.FusedAdamW([p], lr=0.01, betas=(0.9, 0.5), eps=eps, weight_decay=0.0, max_norm=None,
                            state_bits=bits)
        for t in range(1, 4):
            before, g = _np(p), _np(p.grad)
            st = opt.state[p]
            if t == 1:
                m = v = np.zeros(numel)
            elif bits == 32:
                m, v = _np(st["exp_avg"]), _np(st["exp_avg_sq"])
            else:                                     # (bfloat16 ends at 2^-133)
                m, v = A.values(*(x.cpu().numpy() for x in (st["exp_avg"].view(torch.uint8), st["exp_avg_sq"],
                                                            st["exponents"])))
            opt.step()
            assert torch.isfinite(p).all()
            # (m and v in float32, where these numbers have few bits, are the formula's own)
            m, v = (a.astype(np.float64) for a in A.step32(g, m, v, 1.0, (0.9, 0.5)))
            assert v.min() > 0 and v.min() < 2.0**-126
            d = np.sqrt(v) / np.sqrt(1 - 0.5**t) + eps
            move = 0.01 / (1 - 0.9**t) * m / d
            # constants, root, reciprocal and products as in the oracle's step, and p's own rounding
            err = 14 * A.U * np.abs(move) + 3 * A.U * np.abs(before)
            _check(_np(p), before - move, err, torch.float32)


def test_smallest_moments_are_given_back(device):
    """bfloat16 holds what 8 bits do from 2^-130 on, and rounds what is smaller."""
    (p,) = _params([(600,)], torch.float32, device)
    p.grad = torch.exp2(-75 + torch.arange(600, device=device) % 40 / 4.0)
    opt = cl.FusedAdamW([p], betas=(0.9, 0.5), max_norm=None, state_bits=8)
    opt.step()
    st = opt.state[p]
    held = A.values(*(x.cpu().numpy() for x in (st["exp_avg"].view(torch.uint8), st["exp_avg_sq"], st["exponents"])))
    low = 0
    for got, want in zip(opt.moments(), held):
        got, keep = _np(got[0]), np.abs(want) >= 2.0**-130
        low += int(np.sum(~keep & (want != 0)))
        np.testing.assert_array_equal(got[keep], want[keep])
        assert np.all(np.abs(got - want)[~keep] <= 2.0**-134)
    assert low > 100


def test_a_norm_of_nan_scales_nothing(device):
    """NaN stays in its own element; the others step as they would without the clipping."""
    for bits in (32, 8):
        (p,) = _params([(5000,)], torch.float32, device)
        p.grad[17] = float("nan")
        q = copy.deepcopy(p)
        q.grad = p.grad.clone()
        cl.FusedAdamW([p], max_norm=0.5, state_bits=bits).step()
        cl.FusedAdamW([q], max_norm=None, state_bits=bits).step()
        assert torch.isnan(p[17]) and int(torch.isnan(p).sum()) == 1
        keep = torch.arange(5000, device=device) != 17
        assert torch.equal(p[keep], q[keep])


def test_resumes_from_fused_adam(device):
    """Its state dict, which has no weight_decay: the moments, the count and the settings go on."""
    ps = _params([(300, 7), (513,)], torch.float32, device, seed=6)
    adam = cl.FusedAdam(ps, lr=0.02, betas=(0.8, 0.95), eps=1e-6, max_norm=None)
    adam.step()
    adam.step()
    held = [tuple(_np(adam.state[p][k]) for k in ("exp_avg", "exp_avg_sq")) for p in ps]
    opt = cl.FusedAdamW(ps, max_norm=None, weight_decay=0.3)
    opt.load_state_dict(copy.deepcopy(adam.state_dict()))
    before = [_np(p) for p in ps]
    opt.step()
    for p, b, (m, v) in zip(ps, before, held):
        (want, err), _, _ = A.step(b, _np(p.grad), m, v, 3, 1.0, 0.02, (0.8, 0.95), 1e-6, 0.3)
        _check(_np(p), want, err, torch.float32)
        assert float(opt.state[p]["step"]) == 3


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_rounding_at_random(device, dtype):
    """Codes as the random words of the step, the tensors before and the element have them; parameters as
    with the moments before they are rounded."""
    params = _params(SHAPES, dtype, device, seed=3, offset=1)
    with torch.no_grad():
        params[8].grad[300:600] *= 1e-6
        params[9].grad[:20] = 0
    wide, small = params[:3], params[3:]
    betas, lr, eps, decay = (0.9, 0.999), 0.01, 1e-8, 0.1
    opt = cl.FusedAdamW([{"params": wide}, {"params": small, "state_bits": 8}], lr=lr, betas=betas, eps=eps,
                        weight_decay=decay, max_norm=0.5, rounding="random")
    tiles = [-(-p.numel() // 2048) for p in params]
    held = [(np.zeros(p.shape), np.zeros(p.shape)) for p in small]
    for t in range(1, 5):
        scale = A.scale_of([_np(p.grad) for p in params], 0.5)
        before = [_np(p) for p in small]
        opt.step()
        for i, p in enumerate(small):
            g, (m, v) = _np(p.grad), held[i]
            (wp, ep), _, _ = A.step(before[i], g, m, v, t, scale, lr, betas, eps, decay)
            _check(_np(p), wp, ep, dtype)
            words = A.words(t, p.numel(), sum(tiles[:3 + i]))
            codes = A.hold(*A.step32(g, m, v, scale, betas), words)
            st = opt.state[p]
            for name, want in zip(("exp_avg", "exp_avg_sq", "exponents"), codes):
                np.testing.assert_array_equal(st[name].view(torch.uint8).cpu().numpy().reshape(-1), want)
            m, v = A.values(*codes)
            held[i] = m.reshape(p.shape), v.reshape(p.shape)
        for p in params:
            p.grad = (p.grad * (-0.7 if t % 2 else 3.0)).to(dtype)


def test_extremes_rounded_at_random(device):
    p = torch.nn.Parameter(torch.zeros(1024, device=device))
    r = np.random.default_rng(1)
    g = r.standard_normal(1024).astype(np.float32)
    g[5], g[9], g[300] = np.inf, np.nan, -np.inf
    g[512:768] = 2.0**-149
    g[768:] = 1e19
    g[800], g[801] = 1e-19, 0
    p.grad = torch.tensor(g, device=device)
    opt = cl.FusedAdamW([p], betas=(0.9, 0.99), max_norm=None, state_bits=8, rounding="random")
    opt.step()
    with np.errstate(over="ignore", invalid="ignore"):
        cm, cv, powers = A.hold(*A.step32(g, np.zeros(1024), np.zeros(1024), 1.0, (0.9, 0.99)), A.words(1, 1024))
    st = opt.state[p]
    got = st["exp_avg"].view(torch.uint8).cpu().numpy()
    nan = np.array([5, 9, 300])
    assert np.all((got[nan] & 0x7F) == 0x7F)
    keep = np.setdiff1d(np.arange(1024), nan)
    np.testing.assert_array_equal(got[keep], cm[keep])
    np.testing.assert_array_equal(st["exp_avg_sq"].cpu().numpy(), cv)
    np.testing.assert_array_equal(st["exponents"].cpu().numpy(), powers)


def test_random_rounding_in_a_graph(device):
    """Each replay draws its own step's numbers, those of an eager step."""
    eager, graphed = (_params([(5000,), (33, 9)], torch.bfloat16, device) for _ in range(2))
    oe, og = (cl.FusedAdamW(ps, lr=0.01, max_norm=0.3, state_bits=8, rounding="random") for ps in (eager, graphed))
    oe.step()
    og.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        og.step()
    drawn = []
    for _ in range(4):
        oe.step()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(eager, graphed):
            assert torch.equal(p, q)
        for x, y in zip(oe.moments(), og.moments()):
            assert all(torch.equal(s, t) for s, t in zip(x, y))
        drawn.append(og.state[graphed[0]]["exp_avg_sq"].clone())
    assert not any(torch.equal(a, b) for a, b in zip(drawn, drawn[1:]))


@pytest.mark.parametrize("name", ["flat", "shrinks"])
def test_thousands_of_steps_in_8_bits(device, name):
    """Moments and updates next to those of float64.  A held value's relative variance is at most 1/4 (what
    a step changes, times 1/8 of v between codes, summed up), so a mean over 65536 elements is within 6
    deviations, 6 sqrt(1/4 / 65536) = 0.012 (m relative to the root of v); the root's mean is off by 3/8 of
    the variance more."""
    n = 65536
    gen = torch.Generator().manual_seed(8)
    beta2, steps = (0.999, 2500) if name == "flat" else (0.98, 1200)
    sign = torch.randn(n, generator=gen).sign()
    flat = (sign * (0.5 + 1.5 * torch.rand(n, generator=gen))).to(device)
    noise = torch.randn(16, n, generator=gen).to(device)
    p = torch.nn.Parameter(torch.zeros(n, device=device))
    opt = cl.FusedAdamW([p], lr=1.0, betas=(0.9, beta2), eps=1e-12, weight_decay=0.0, max_norm=None,
                        state_bits=8, rounding="random")
    fm = fv = torch.zeros(n, dtype=torch.float64, device=device)
    for t in range(1, steps + 1):
        p.grad = flat if name == "flat" else noise[t % 16] * (1.0 if t < 400 else 0.1)
        fm, fv = 0.9 * fm + 0.1 * p.grad.double(), beta2 * fv + (1 - beta2) * p.grad.double()**2
        if t == steps:
            p.data.zero_()
        opt.step()
    m, v = (x[0].double() for x in opt.moments())
    assert abs(float(v.mean() / fv.mean()) - 1) < 0.012
    assert abs(float(((m - fm) * fm.sign()).mean() / fv.mean().sqrt())) < 0.012
    want = fm / (1 - 0.9**steps) / (fv / (1 - beta2**steps)).sqrt()
    assert abs(float(p.abs().mean().double() / want.abs().mean()) - 1) < 0.012 + 3 / 8 / 4
