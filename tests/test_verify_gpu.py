"""verify_drafts against the oracle: tokens and counts equal, log-probabilities in float64."""
import numpy as np
import pytest
import torch

import compactlogic_amd as cl
from oracle import verify_np as V

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]
# (sequences, drafts, classes): one chunk of a row and its borders, several; more positions than a
# round of tests takes in either path
SHAPES = [(1, 0, 1), (3, 0, 10), (5, 1, 2), (256, 4, 10), (7, 3, 63), (4, 2, 1000), (5, 9, 512), (3, 2, 513), (3, 2, 4096),
          (3, 2, 4097), (3, 5, 8191), (3, 5, 8192),
          (3, 2, 8193), (2, 3, 20011), (1, 7, 131072), (2, 37, 8200), (5, 41, 50)]


def _inputs(shape, dtype, device, seed, noise=0.5):
    s, k, v = shape
    gen = torch.Generator().manual_seed(seed)
    logits = (torch.randn((s, k + 1, v), generator=gen) * 2.5).to(dtype)
    draft = (logits[:, :k].double() + noise * torch.randn((s, k, v), generator=gen)).to(dtype)
    z = draft.double()
    tokens = (z - torch.log(-torch.log(torch.rand(z.shape, generator=gen, dtype=torch.float64)))).argmax(2) \
        if k else torch.zeros((s, 0), dtype=torch.int64)
    uniforms = torch.rand((s, k + 1), generator=gen)
    return [t.to(device) for t in (logits, tokens, draft, uniforms)]


def _check(got, logits, tokens, draft, uniforms, ignore=-100):
    np64 = lambda t: None if t is None else t.double().cpu().numpy()
    want = V.verify(np64(logits), tokens.cpu().numpy(), np64(draft), np64(uniforms), ignore)
    out, accepted, lp = got
    k = tokens.shape[1]
    assert out.dtype == accepted.dtype == torch.int64 and out.shape == lp.shape == (len(tokens), k + 1)
    np.testing.assert_array_equal(accepted.cpu().numpy(), want[1])
    np.testing.assert_array_equal(out.cpu().numpy(), want[0])
    # a sum of V terms in fp32, of which each partial sum is rounded (over lanes, then in some 40
    # steps each), exponentials within 8e-7, then the result's rounding
    wide = torch.float64 if logits.dtype == torch.float64 else torch.float32
    assert lp.dtype == wide
    tol = 1e-13 if wide == torch.float64 else 8e-7 + 60 * 2.0**-24
    rel = torch.finfo(wide).eps / 2
    np.testing.assert_allclose(lp.double().cpu().numpy(), want[2], rtol=rel * 1.01 + 1e-15, atol=tol)
    return want


@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
def test_matches_oracle(device, dtype, with_draft):
    for i, shape in enumerate(SHAPES):
        print(shape, flush=True)
        logits, tokens, draft, uniforms = _inputs(shape, dtype, device, i)
        if not with_draft:
            # sure of its tokens: the target's likeliest, so that some are accepted
            tokens, draft = logits[:, :shape[1]].argmax(2), None
        got = cl.verify_drafts(logits, tokens, draft, uniforms)
        want = _check(got, logits, tokens, draft, uniforms)
        if shape == (256, 4, 10):
            assert set(want[1]) == {0, 1, 2, 3, 4}    # every outcome


@pytest.mark.parametrize("vocab", [33, 9000])
def test_shorter_drafts(device, vocab):
    """ignore_index ends a sequence's drafts, at the first of them; other tokens outside are refused."""
    logits, tokens, draft, uniforms = _inputs((12, 6, vocab), torch.float32, device, 3, noise=0.1)
    for s in range(6):
        tokens[s, s] = -100
    tokens[1, 3] = 5
    tokens[7, 0], tokens[8, 2], tokens[9, 1] = vocab, -1, -(2**62)
    for q in (draft, None):
        want = _check(cl.verify_drafts(logits, tokens, q, uniforms), logits, tokens, q, uniforms)
        assert all(want[1][s] <= s for s in range(6))
    # logits behind the end are not looked at
    for s in range(6):
        logits[s, s + 1:] = float("nan")
        draft[s, s:] = float("nan")
    want = _check(cl.verify_drafts(logits, tokens, draft, uniforms), logits, tokens, draft, uniforms)
    assert np.isfinite(want[2][:6]).all()
    tokens[tokens == -100] = 7777
    _check(cl.verify_drafts(logits, tokens, draft, uniforms, ignore_index=7777), logits, tokens, draft, uniforms,
           7777)


@pytest.mark.parametrize("vocab", [40, 10007])
def test_masked_and_broken_logits(device, vocab):
    logits, tokens, draft, uniforms = _inputs((16, 3, vocab), torch.float32, device, 4, noise=0.1)
    logits[0, :, ::2] = draft[0, :, ::2] = float("-inf")    # masked in both
    logits[1, :, 1::2] = float("-inf")                      # the draft offers what the target forbids
    tokens[1] = 1
    logits[2, 1] = float("-inf")                            # no token at all
    logits[3, 1, 3] = float("nan")
    logits[4, 0, 3] = float("inf")
    draft[5, 0, 3] = float("nan")                           # refused, then the target's own
    logits[6] = torch.finfo(torch.float32).min              # even, at the type's lowest value
    logits[7, :, 1:] = float("-inf")                        # one token left
    draft[8, 1] = float("-inf")
    logits[9, :, :-1] = float("-inf")                       # the last one
    for q in (draft, None):
        want = _check(cl.verify_drafts(logits, tokens, q, uniforms), logits, tokens, q, uniforms)
        assert want[1][1] == 0 and np.isnan(want[2][4]).any() and want[0][4, want[1][4]] == -100
        assert want[0][7, want[1][7]] == 0 and want[0][9, want[1][9]] == vocab - 1


@pytest.mark.parametrize("vocab", [10, 20000])
def test_ends_of_the_random_numbers(device, vocab):
    logits, tokens, draft, _ = _inputs((40, 3, vocab), torch.float32, device, 5)
    logits[::2, :, 0] = float("-inf")
    logits[::3, :, -1] = float("-inf")
    below = float(np.nextafter(np.float32(1), np.float32(0)))
    for u in (0.0, below):
        uniforms = torch.full((40, 4), u, device=device)
        _check(cl.verify_drafts(logits, tokens, draft, uniforms), logits, tokens, draft, uniforms)
        wide = uniforms.double()
        _check(cl.verify_drafts(logits, tokens, draft, wide), logits, tokens, draft, wide)
    # the likeliest token 740 above the others: probabilities below the smallest normal fp64 number
    far = torch.full((40, 4, vocab), -740.0, device=device)
    far[:, :, vocab // 2] = 0.0
    none = torch.full((40, 3), -100, dtype=torch.int64, device=device)
    uniforms = torch.zeros((40, 4), device=device)
    want = _check(cl.verify_drafts(far, none, None, uniforms), far, none, None, uniforms)
    assert (want[0][:, 0] == 0).all()
    # a draft that is the target: every token accepted below 1, and nothing above it to draw from at 1
    uniforms = torch.full((40, 4), below, device=device)
    tokens = draft.argmax(2)
    out, accepted, _ = cl.verify_drafts(draft[:, [0, 1, 2, 0]], tokens, draft, uniforms)
    assert (accepted == 3).all() and torch.equal(out[:, :3], tokens)
    uniforms[:, :3] = 1.0
    same = draft[:, [0, 1, 2, 0]].contiguous()
    want = _check(cl.verify_drafts(same, tokens, draft, uniforms), same, tokens, draft, uniforms)
    assert (want[1] == 0).all()


def test_many_thresholds_of_one_row(device):
    """Draws along the whole row: each token where its share of the numbers lies, in both paths."""
    for vocab in (100, 8193):
        gen = torch.Generator().manual_seed(6)
        z = torch.randn(vocab, generator=gen, dtype=torch.float64)
        u = torch.arange(1000, dtype=torch.float64) / 1000
        out, _, _ = cl.verify_drafts(z.to(device).expand(1000, 1, vocab),
                                     torch.zeros((1000, 0), dtype=torch.int64, device=device), None,
                                     u[:, None].to(device))
        sums = torch.cumsum(torch.softmax(z, 0), 0)
        want = torch.searchsorted(sums, u * sums[-1], right=True)
        assert torch.equal(out[:, 0].cpu(), want)


def test_layouts_and_leading_dimensions(device):
    for vocab in (37, 9001):
        logits, tokens, draft, uniforms = _inputs((6, 2, vocab), torch.bfloat16, device, 7)
        want = cl.verify_drafts(logits, tokens, draft, uniforms)
        lead = cl.verify_drafts(logits.view(2, 3, 3, vocab), tokens.view(2, 3, 2), draft.view(2, 3, 2, vocab),
                                uniforms.view(2, 3, 3))
        one = cl.verify_drafts(logits[4], tokens[4], draft[4], uniforms[4])
        assert lead[0].shape == (2, 3, 3) and lead[1].shape == (2, 3) and one[1].shape == ()
        for a, b, c in zip(want, lead, one):
            assert torch.equal(a.reshape(-1), b.reshape(-1)) and torch.equal(a[4], c)
        padded = torch.zeros((6, 4, vocab + 3), dtype=logits.dtype, device=device)[:, 1:, 1:vocab + 1].copy_(logits)
        turned = logits.permute(2, 1, 0).contiguous().permute(2, 1, 0)
        by_place = draft.transpose(0, 1).contiguous().transpose(0, 1)
        for z, q in ((padded, by_place), (turned, draft)):
            got = cl.verify_drafts(z, tokens.t().contiguous().t(), q, uniforms.t().contiguous().t())
            assert all(torch.equal(a, b) for a, b in zip(want, got))
        shared = logits[:1].expand(6, 3, vocab)
        _check(cl.verify_drafts(shared, tokens, draft, uniforms), shared, tokens, draft, uniforms)
    empty = cl.verify_drafts(logits[:0], tokens[:0], draft[:0], uniforms[:0])
    assert [t.shape for t in empty] == [(0, 3), (0,), (0, 3)]


def test_distribution(device):
    """Of n sequences the share of each first token lies within 5 standard deviations of the target's
    probability, whatever the draft."""
    n = 200_000
    gen = torch.Generator(device=device).manual_seed(8)
    p = torch.tensor([0.5, 0.2, 0.25, 0.05], device=device)
    q = torch.tensor([0.1, 0.6, 0.1, 0.2], device=device)
    tokens = torch.multinomial(q, n, replacement=True, generator=gen)[:, None]
    u = torch.rand((n, 2), generator=gen, device=device)
    out, accepted, _ = cl.verify_drafts(p.log().expand(n, 2, 4), tokens, q.log().expand(n, 1, 4), u)
    for draws in (out[:, 0], out[accepted == 1, 1]):
        share = torch.bincount(draws, minlength=4) / len(draws)
        assert ((share - p).abs() <= 5 * (p * (1 - p) / len(draws)).sqrt()).all()


@pytest.mark.parametrize("vocab", [50, 9000])
def test_graph_replays_like_eager(device, vocab):
    args = _inputs((9, 3, vocab), torch.float32, device, 9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cl.verify_drafts(*args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = cl.verify_drafts(*args)
    for k in range(4):
        for t, new in zip(args, _inputs((9, 3, vocab), torch.float32, device, 10 + k)):
            t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, cl.verify_drafts(*args)))


def test_another_stream_and_requires_grad(device):
    logits, tokens, draft, uniforms = _inputs((9, 3, 20000), torch.float32, device, 20)
    want = cl.verify_drafts(logits, tokens, draft, uniforms)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = cl.verify_drafts(logits.requires_grad_(), tokens, draft, uniforms)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and not got[2].requires_grad


def test_more_than_32_bits_of_logits(device):
    s, k, v = 601, 3, 1_000_003               # 2.4e9 logits
    logits = torch.zeros((s, k + 1, v), dtype=torch.bfloat16, device=device)
    tokens = torch.full((s, k), 17, dtype=torch.int64, device=device)
    logits[-1, 0, 17] = logits[-1, 1, v - 1] = 60.0
    tokens[-1, 1] = v - 1
    logits[-1, 2, v - 2] = 60.0
    uniforms = torch.full((s, k + 1), 0.5, device=device)
    out, accepted, lp = cl.verify_drafts(logits, tokens, None, uniforms)
    assert out[-1].tolist() == [17, v - 1, v - 2, -100] and int(accepted[-1]) == 2
    assert (accepted[:-1] == 0).all() and (out[:-1, 0] == (v + 1) // 2).all()   # all but 17, evenly
    assert float((lp[:-1, 0] + np.log(v)).abs().max()) < 1e-5


def test_refusals(device):
    logits, tokens, draft, uniforms = _inputs((2, 3, 5), torch.float32, device, 0)
    for bad, what in ((dict(z=logits.long()), "dtype"), (dict(z=logits[0, 0]), "drafts"),
                      (dict(z=logits[:, :0]), "drafts"), (dict(z=logits[..., :0]), "classes"),
                      (dict(t=tokens.int()), "draft_tokens"), (dict(t=tokens[:, :2]), "draft_tokens"),
                      (dict(u=uniforms.half()), "uniforms"), (dict(u=uniforms[:, :3]), "uniforms"),
                      (dict(q=draft.half()), "draft_logits"), (dict(q=draft[:, :2]), "draft_logits"),
                      (dict(q=draft.cpu()), "draft_logits"), (dict(t=tokens.cpu()), "HIP device")):
        args = {"z": logits, "t": tokens, "q": draft, "u": uniforms, **bad}
        with pytest.raises(RuntimeError, match=what):
            cl.verify_drafts(args["z"], args["t"], args["q"], args["u"])
    with pytest.raises(TypeError, match="draft_logits"):
        cl.verify_drafts(logits, tokens, 1.0, uniforms)
