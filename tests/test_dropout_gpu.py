"""Dropout against the oracle: the mask bit by bit, values, gradients, layouts, graphs."""
import numpy as np
import pytest
import torch
import torch.utils.checkpoint

import compactlogic_amd as cl
from oracle import dropout_np as D

pytestmark = pytest.mark.gpu

SEED, OFFSET = 0x1234567890ABCDEF, 0xFEDCBA9876543210
DTYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]
SHAPES = [(1, 1), (1, 7), (7, 1), (3, 8), (5, 9), (64, 15), (65, 64), (33, 257), (2, 4099),
          (1027, 24), (300, 1001)]


def _lay(t, layout):
    """t with its values, lying as `layout` says."""
    rows, cols = t.shape
    if layout == "rows":
        return t.clone()
    if layout == "columns":
        return t.t().contiguous().t()
    if layout == "padded":                # rows 3 elements apart, off 16 bytes
        return torch.zeros((rows, cols + 3), dtype=t.dtype, device=t.device)[:, 1:cols + 1].copy_(t)
    if layout == "padded columns":
        return torch.zeros((cols, rows + 5), dtype=t.dtype,
                           device=t.device)[:, 1:rows + 1].t().copy_(t)
    assert layout == "strided"            # neither dimension contiguous
    return torch.zeros((rows, 2 * cols), dtype=t.dtype, device=t.device)[:, ::2].copy_(t)


def _close(got, ref, dtype, exact):
    """Kept elements are one product by the scale, in fp32 (fp64), and one rounding: scale, product
    and storage round by half a step each; 16-bit results may round a product that is 2^-23 off."""
    got = got.double().cpu().numpy()
    if exact:
        np.testing.assert_array_equal(got, ref)
        return
    half = torch.finfo(dtype).eps / 2
    wide = 2.0**-53 if dtype == torch.float64 else 2.0**-24
    tiny = torch.finfo(dtype).smallest_normal * half * 2
    assert np.all(np.abs(got - ref) <= np.abs(ref) * (half + 2 * wide) * 1.001 + tiny)


@pytest.mark.parametrize("layout", ["rows", "columns", "padded", "padded columns", "strided"])
@pytest.mark.parametrize("fill", [None, 0.5])
@pytest.mark.parametrize("dtype", DTYPES)
def test_matches_oracle(device, dtype, fill, layout):
    for i, (rows, cols) in enumerate(SHAPES):
        g = torch.Generator().manual_seed(i)
        p = [0.1, 0.5, 0.9][i % 3]
        x = _lay(torch.rand((rows, cols), generator=g).to(dtype).to(device), layout)
        gy = _lay(torch.randn((rows, cols), generator=g).to(dtype).to(device), layout)
        xn, gn = x.double().cpu().numpy(), gy.double().cpu().numpy()
        x.requires_grad_()
        y = cl.dropout(x, p, SEED, OFFSET, fill=fill)
        (gx,) = torch.autograd.grad(y, x, gy)
        assert y.shape == x.shape and y.dtype == dtype and gx.dtype == dtype
        _close(y.detach(), D.dropout(xn, p, SEED, OFFSET, fill), dtype, fill is not None)
        _close(gx, D.dropout(gn, p, SEED, OFFSET, None if fill is None else 0.0), dtype,
               fill is not None)
        if layout == "columns":
            assert y.t().is_contiguous() and gx.t().is_contiguous()
        # the same mask from the device's state
        rng = torch.tensor([SEED, OFFSET - 2**64], dtype=torch.int64, device=device)
        assert torch.equal(cl.dropout(x, p, rng, fill=fill), y)


def test_mask_is_a_function_of_the_place(device):
    """Equal masks in every layout, type and number of leading dimensions; another offset or seed
    gives another mask."""
    ones = torch.ones(60, 77, device=device)
    y = cl.dropout(ones, 0.5, SEED, 3, fill=0.0)
    assert torch.equal(y, cl.dropout(ones.t().contiguous().t(), 0.5, SEED, 3, fill=0.0))
    assert torch.equal(y, cl.dropout(ones.bfloat16(), 0.5, SEED, 3, fill=0.0).float())
    assert torch.equal(y, cl.dropout(ones.view(60, 7, 1, 11), 0.5, SEED, 3, fill=0.0).view(60, 77))
    last = ones.view(60, 7, 11).permute(1, 2, 0).contiguous().permute(2, 0, 1)  # feature-major
    assert torch.equal(y, cl.dropout(last, 0.5, SEED, 3, fill=0.0).reshape(60, 77))
    odd = ones.view(60, 7, 11).transpose(1, 2)                                   # copied
    assert torch.equal(cl.dropout(odd, 0.5, SEED, 3, fill=0.0).reshape(60, 77), y)
    assert torch.equal(y[:1, 0:1].reshape(()), cl.dropout(ones[0, 0], 0.5, SEED, 3, fill=0.0))
    assert torch.equal(y[0], cl.dropout(ones[0], 0.5, SEED, 3, fill=0.0))
    assert torch.equal(y[:17, :33], cl.dropout(ones[:17, :33], 0.5, SEED, 3, fill=0.0))
    assert not torch.equal(y, cl.dropout(ones, 0.5, SEED, 4, fill=0.0))
    assert not torch.equal(y, cl.dropout(ones, 0.5, SEED + 1, 3, fill=0.0))


def test_extremes(device):
    x = torch.tensor([[1.0, float("nan"), float("inf"), -0.0]], device=device)
    x = x.expand(50, 4).contiguous()
    assert cl.dropout(x, 0.0, 1) is x and cl.dropout(x, 2.0**-18, 1) is x
    assert torch.equal(cl.dropout(x, 1.0, 1), torch.zeros_like(x))     # NaN and inf go as well
    assert torch.equal(cl.dropout(x, 1.0, 1, fill=0.5), torch.full_like(x, 0.5))
    keep = torch.from_numpy(D.keep_mask(50, 4, 0.5, 1)).to(device)
    y = cl.dropout(x, 0.5, 1)
    assert torch.equal(y.isnan(), keep & x.isnan()) and torch.equal(y.isinf(), keep & x.isinf())
    empty = torch.empty(0, 5, device=device)
    assert cl.dropout(empty, 0.5, 1) is empty
    row = torch.rand(1, 40, device=device).expand(30, 40)              # rows of stride 0
    assert torch.equal(cl.dropout(row, 0.5, 1), cl.dropout(row.contiguous(), 0.5, 1))
    e = row[:1].clone().requires_grad_()
    (g,) = torch.autograd.grad(cl.dropout(e.expand(30, 40), 0.5, 1).sum(), e)
    ref = D.keep_mask(30, 40, 0.5, 1).sum(0) * 2.0
    np.testing.assert_array_equal(g[0].cpu().numpy(), ref)             # whole numbers: exact


def test_refusals(device):
    x = torch.rand(4, 8, device=device)
    with pytest.raises(ValueError, match="probability"):
        cl.dropout(x, 1.5, 1)
    with pytest.raises(RuntimeError, match="dtype"):
        cl.dropout(x.long(), 0.5, 1)
    for seed in (torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=torch.int64, device=device),
                 torch.zeros(2, device=device)):
        with pytest.raises(RuntimeError, match="seed"):
            cl.dropout(x, 0.5, seed)
    with pytest.raises(ValueError, match="offset"):
        cl.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64, device=device), 3)
    with pytest.raises(RuntimeError, match="rng must be"):
        cl.Dropout(0.5)(x)                                             # the module is on the host
    # the state of a mask must not change before its backward
    rng = torch.tensor([1, 2], device=device)
    y = cl.dropout(x.requires_grad_(), 0.5, rng).sum()
    rng += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_gradient_of_the_gradient(device):
    """d/dx of sum over (d/dx of sum keep(x^3)) = keep 6 x, scaled once by each pass; the scale 2
    and the products of small whole numbers are exact."""
    x = torch.arange(32, device=device, dtype=torch.float32).view(4, 8).requires_grad_()
    keep = torch.from_numpy(D.keep_mask(4, 8, 0.5, 1)).to(device).float()
    for fill, scale in ((None, 2.0), (0.5, 1.0)):
        y = cl.dropout(x * x * x, 0.5, 1, fill=fill)
        (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
        assert torch.equal(g, 3 * x * x * keep * scale)
        (h,) = torch.autograd.grad(g.sum(), x)
        assert torch.equal(h, 6 * x * keep * scale)
        # through the upstream gradient too
        up = torch.ones(4, 8, device=device, requires_grad=True)
        (g,) = torch.autograd.grad(cl.dropout(x, 0.5, 1, fill=fill), x, up, create_graph=True)
        assert torch.equal(torch.autograd.grad(g.sum(), up)[0], keep * scale)


def test_module_draws_new_masks_and_resumes(device):
    m = cl.Dropout(0.5, seed=11).to(device)
    x = torch.ones(32, 100, device=device)
    a, b = m(x), m(x)
    for k, y in enumerate((a, b)):
        np.testing.assert_array_equal(y.cpu().numpy(), 2.0 * D.keep_mask(32, 100, 0.5, 11, k))
    other = cl.Dropout(0.5, seed=99).to(device)
    other.load_state_dict(m.state_dict())
    assert torch.equal(other(x), m(x)) and m.rng.tolist() == [11, 3]
    # gradient through the mask of its own call, with another call between
    z = x.clone().requires_grad_()
    y = m(z)
    m(x)
    y.sum().backward()
    assert torch.equal(z.grad, y.detach())
    # a mask asked for again: the offset is the number of the call
    assert torch.equal(cl.dropout(x, 0.5, 11, 1), b)
    bits = cl.PackBitsTensor(x > 0, 64)
    assert m(bits) is bits and m.eval()(x) is x


def test_captured_step_draws_a_new_mask_each_replay(device):
    m = cl.Dropout(0.5, seed=5).to(device)
    x = torch.ones(40, 64, device=device, requires_grad=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(m(x).sum(), x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m(x)
        (g,) = torch.autograd.grad(y.sum(), x)
    for k in range(1, 5):
        torch.randn(1000, device=device).sum()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ref = 2.0 * D.keep_mask(40, 64, 0.5, 5, k)
        np.testing.assert_array_equal(y.detach().cpu().numpy(), ref)
        np.testing.assert_array_equal(g.cpu().numpy(), ref)


def test_other_streams(device):
    x = torch.ones(64, 1000, device=device)
    ref = cl.dropout(x, 0.5, 7)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = cl.dropout(x, 0.5, 7)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, ref)


def test_network_with_dropout_matches_its_layers(device):
    """Between logic layers in training; left out of packed and circuit inference."""
    torch.manual_seed(0)
    drop = cl.Dropout(0.25, fill=0.5, seed=3)
    layers = [cl.LogicLayer(64, 200), drop, cl.LogicLayer(200, 200), cl.GroupSum(10, 2.0)]
    net = torch.nn.Sequential(*layers).to(device)
    x = (torch.rand(96, 64, device=device) < 0.5).float()
    labels = torch.randint(0, 10, (96,), device=device)
    loss = cl.sequential_cross_entropy(net, x, labels)
    loss.backward()
    h = net[0](x)
    keep = torch.from_numpy(D.keep_mask(96, 200, 0.25, 3, 0)).to(device)
    ref = net[3].cross_entropy(net[2](torch.where(keep, h, 0.5)), labels)
    grads = [p.grad for p in net.parameters()]
    # the same values through the same kernels, the loss by another order of sums
    assert abs(float(loss) - float(ref)) <= 1e-5 * abs(float(ref))
    for g, r in zip(grads, torch.autograd.grad(ref, list(net.parameters()))):
        assert torch.allclose(g, r, rtol=1e-4, atol=1e-6)
    plain = torch.nn.Sequential(net[0], net[2], net[3])
    for m in (net[0], net[2]):
        m.freeze()
    net.eval()
    bits = x.bool()
    want = plain(cl.PackBitsTensor(bits, 64))
    assert torch.equal(net(cl.PackBitsTensor(bits, 64)), want)
    assert torch.equal(cl.PackedNetwork(net)(cl.PackBitsTensor(bits, 64)), want)
    c = cl.circuit.extract_circuit(net)
    assert c.k == 10 and len(c.gates) == 2


@pytest.mark.parametrize("layout", ["rows", "columns"])
def test_large_tensors(device, layout):
    """First, middle and last rows of tensors past 32 bits, against the oracle's counters."""
    if layout == "rows":                  # 2^31 blocks and some, one each for a thread
        rows, cols = 262145, 65536
        x = torch.ones((rows, cols), dtype=torch.bfloat16, device=device)
    else:                                 # 2^32 elements and some
        rows, cols = 70000, 65537
        x = torch.ones((cols, rows), dtype=torch.bfloat16, device=device).t()
    y = cl.dropout(x, 0.5, SEED, OFFSET, fill=0.0)
    for r in (0, rows // 2, rows - 1):
        blocks = -(-cols // 8)
        counter = np.zeros((blocks, 4), dtype=np.uint64)
        counter[:, 0], counter[:, 1] = np.arange(blocks), r
        counter[:, 2], counter[:, 3] = OFFSET & 0xFFFFFFFF, OFFSET >> 32
        words = D.philox(counter, np.array([SEED & 0xFFFFFFFF, SEED >> 32], dtype=np.uint64))
        halves = np.stack((words & 0xFFFF, words >> 16), -1).reshape(-1)[:cols]
        np.testing.assert_array_equal(y[r].float().cpu().numpy(), (halves >= 32768) * 1.0)


def test_threads_past_32_bits(device):
    """2^32 generator blocks and some (69 GB), a thread each: the first and last rows against the
    oracle's counters."""
    rows, cols = (1 << 20) + 1, 32768
    x = torch.ones((1, cols), dtype=torch.bfloat16, device=device).expand(rows, cols)
    y = cl.dropout(x, 0.5, SEED, OFFSET, fill=0.0)
    counter = np.zeros((cols // 8, 4), dtype=np.uint64)
    counter[:, 0] = np.arange(cols // 8)
    counter[:, 2], counter[:, 3] = OFFSET & 0xFFFFFFFF, OFFSET >> 32
    for r in (0, rows // 2, rows - 2, rows - 1):
        counter[:, 1] = r
        words = D.philox(counter, np.array([SEED & 0xFFFFFFFF, SEED >> 32], dtype=np.uint64))
        halves = np.stack((words & 0xFFFF, words >> 16), -1).reshape(-1)
        np.testing.assert_array_equal(y[r].float().cpu().numpy(), (halves >= 32768) * 1.0)
    del y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("reentrant", [False, True])
def test_module_in_a_recomputed_segment(device, reentrant):
    """The module would draw another mask there and is refused; a mask taken before the segment
    gives what the segment gives without recomputation."""
    x = torch.rand(33, 70, device=device, requires_grad=True)
    drop = cl.Dropout(0.5, seed=3).to(device)

    def segment(h):
        return drop(h * h).sum()

    y = torch.utils.checkpoint.checkpoint(segment, x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="next_rng"):
        y.backward()
    assert drop.rng.tolist() == [3, 1]

    rng = drop.next_rng()

    def masked(h):
        return cl.dropout(h * h, drop.p, rng, fill=drop.fill).sum()

    (want,) = torch.autograd.grad(masked(x), x)
    x.grad = None
    torch.utils.checkpoint.checkpoint(masked, x, use_reentrant=reentrant).backward()
    assert torch.equal(x.grad, want) and drop.rng.tolist() == [3, 2]
    keep = D.keep_mask(33, 70, 0.5, 3, 1)
    assert np.array_equal(want.cpu().numpy() != 0, keep & (x.detach().cpu().numpy() != 0))
