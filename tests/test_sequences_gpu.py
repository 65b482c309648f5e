"""Sequences as a policy uses them: a layer of latches and its state, drafted actions verified, the
policy loss on what was drawn, the optimizer step, against the same in plain torch and float64."""
import copy

import numpy as np
import pytest
import torch

import compactlogic_amd as cl
from oracle import adamw_np as A
from oracle import verify_np as V

pytestmark = pytest.mark.gpu

BATCH, DRAFTS, INPUTS, HIDDEN, ACTIONS, TAU = 24, 5, 20, 40, 4, 3.0


class Policy(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.memory = cl.LogicRecurrence(INPUTS, HIDDEN)
        self.head = cl.LogicLayer(HIDDEN, 12 * ACTIONS)
        self.scores = cl.GroupSum(ACTIONS, TAU)

    def forward(self, x, state=None):
        h, state = self.memory(x, state, return_state=True)
        y = self.head(h.reshape(-1, HIDDEN))
        return self.scores(y).reshape(*x.shape[:2], ACTIONS), state


def _plain(policy, x, state):
    """The scores with the latches walked step by step in torch, in float64."""
    flat = x.reshape(-1, INPUTS)
    gate, data = (f(flat).double().reshape(*x.shape[:2], HIDDEN)
                  for f in (policy.memory.gate, policy.memory.data))
    h, steps = state.double(), []
    for t in range(x.shape[1]):
        h = gate[:, t] * h + (1 - gate[:, t]) * data[:, t]
        steps.append(h)
    h = torch.stack(steps, 1).reshape(-1, HIDDEN).float()
    y = policy.head(h).double()
    return y.reshape(*x.shape[:2], ACTIONS, 12).sum(3) / TAU


def _world(device):
    torch.manual_seed(0)
    policy = Policy().to(device)
    draft = copy.deepcopy(policy).eval()          # the discretized network drafts
    gen = torch.Generator(device=device).manual_seed(1)
    x = (torch.rand((BATCH, DRAFTS + 1, INPUTS), generator=gen, device=device) < 0.5).float()
    state = torch.rand((BATCH, HIDDEN), generator=gen, device=device)
    noise = torch.rand((BATCH, DRAFTS, ACTIONS), generator=gen, device=device)
    uniforms = torch.rand((BATCH, DRAFTS + 1), generator=gen, device=device)
    return policy, draft, x, state, noise, uniforms


def _rollout(policy, draft, x, state, noise, uniforms):
    """Actions drafted one by one, then verified by one evaluation of the policy."""
    with torch.no_grad():
        scores, tokens, s = [], [], state
        for t in range(DRAFTS):
            z, s = draft(x[:, t:t + 1], s)
            scores.append(z)
            tokens.append((z[:, 0] - torch.log(-torch.log(noise[:, t]))).argmax(1))
        drafted, tokens = torch.cat(scores, 1), torch.stack(tokens, 1)
        target, _ = policy(x, state)
        return cl.verify_drafts(target, tokens, drafted, uniforms), target, tokens, drafted


def _loss(policy, x, state, actions, old, adv):
    z, _ = policy(x, state)
    return cl.policy_loss(z, actions, old, adv)


@pytest.mark.parametrize("bits", [32, 8])
def test_rollout_and_step(device, bits):
    policy, draft, x, state, noise, uniforms = _world(device)
    (actions, accepted, lp), target, tokens, drafted = _rollout(policy, draft, x, state, noise, uniforms)
    want = V.verify(target.double().cpu().numpy(), tokens.cpu().numpy(), drafted.double().cpu().numpy(),
                    uniforms.cpu().numpy())
    np.testing.assert_array_equal(actions.cpu().numpy(), want[0])
    np.testing.assert_array_equal(accepted.cpu().numpy(), want[1])
    # (sums of four exponentials in fp32)
    np.testing.assert_allclose(lp.cpu().numpy(), want[2], rtol=1e-6, atol=2e-6)
    assert len(set(want[1])) > 2
    # the policy that acted is the one that is trained: every ratio is 1 up to rounding
    adv = torch.randn(lp.shape, generator=torch.Generator().manual_seed(2)).to(device)
    loss = _loss(policy, x, state, actions, lp, adv)
    loss.backward()
    counted = actions != -100
    np.testing.assert_allclose(float(loss.detach()), -float(adv[counted].double().mean()), rtol=1e-4, atol=1e-5)
    grads = [p.grad.clone() for p in policy.parameters()]
    z = _plain(policy, x, state)
    logp = torch.log_softmax(z, 2).gather(2, actions.clamp(min=0)[..., None])[..., 0]
    ratio = torch.exp(logp - lp.double())
    gain = torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv)
    ref = torch.autograd.grad(-gain[counted].mean(), list(policy.parameters()))
    for a, b in zip(grads, ref):                  # sums over 144 steps' fp32 terms on both sides
        np.testing.assert_allclose(a.double().cpu().numpy(), b.double().cpu().numpy(), rtol=1e-4,
                                   atol=1e-7)
    before = [p.detach().double().cpu().numpy() for p in policy.parameters()]
    g = [t.double().cpu().numpy() for t in grads]
    norm = np.sqrt(sum(float(np.sum(d * d)) for d in g))
    opt = cl.FusedAdamW(policy.parameters(), lr=0.01, weight_decay=0.1, max_norm=norm / 2, state_bits=bits)
    scale = A.scale_of(g, norm / 2)
    opt.step()
    for p, old, d in zip(policy.parameters(), before, g):
        (new, err), _, _ = A.step(old, d, 0 * d, 0 * d, 1, scale, 0.01, (0.9, 0.999), 1e-8, 0.1)
        got = p.detach().double().cpu().numpy()
        assert np.all(np.abs(got - new) <= err * 1.001 + np.abs(new) * 2.0**-24)


def test_training_step_in_a_graph(device):
    """Latches, loss, backward and step in one captured graph, replayed among eager ones."""
    steps = []
    for graphed in (False, True):
        policy, draft, x, state, noise, uniforms = _world(device)
        (actions, _, lp), *_ = _rollout(policy, draft, x, state, noise, uniforms)
        adv = torch.randn(lp.shape, generator=torch.Generator().manual_seed(2)).to(device)
        opt = cl.FusedAdamW(policy.parameters(), lr=0.02, state_bits=8)

        def step():
            policy.zero_grad(set_to_none=True)
            loss = _loss(policy, x, state, actions, lp, adv)
            loss.backward()
            opt.step()
            return loss.detach()

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        if graphed:
            policy.zero_grad(set_to_none=True)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                loss = step()
        seen = []
        for k in range(4):
            x.copy_((x + (k % 2)) % 2)
            if graphed:
                graph.replay()
                torch.cuda.synchronize()
                seen.append(float(loss))
            else:
                seen.append(float(step()))
        steps.append((seen, [p.detach().clone() for p in policy.parameters()]))
    assert steps[0][0] == steps[1][0]
    assert all(torch.equal(a, b) for a, b in zip(steps[0][1], steps[1][1]))
