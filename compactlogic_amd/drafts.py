"""Drawing actions or tokens, with or without drafts, on the HIP kernels.  No counterpart in the
reference.

A cheap network (a discretized one, a smaller one) drafts a few tokens, and the target's logits behind
each of them, which one evaluation gives for all, decide which are kept; what results is distributed
as the target's own tokens are.  Tokens and log-probabilities come out as `policy_loss` takes them.
"""
from __future__ import annotations

import torch

from . import _native
from . import difflogic_hip as _dl


def verify_drafts(logits, draft_tokens, draft_logits, uniforms, ignore_index: int = -100):
    """Keeps the drafted tokens that the target's probabilities bear out, and draws one more.

    logits [..., K + 1, V]: the target's, behind each of the K drafted tokens' predecessors and behind
    the last one; draft_tokens int64 [..., K]; draft_logits [..., K, V]: what they were drawn from, or
    None for a draft that was sure of each (a greedy one: probability 1); uniforms [..., K + 1]:
    random numbers in [0, 1), float32 or float64.  With p and q the softmax of a position's logits, its
    token x is accepted while u q(x) < p(x).  At the first one that is not, a token is drawn from
    max(p - q, 0), and behind the last one from p: by the last uniform number r, the first token whose
    sum of weights up to it is above r times their whole sum.  K = 0 draws one token of each row.

    The first draft token that is ignore_index ends its sequence's drafts.  Another one outside of the
    V classes has probability 0 and is refused.  Logits of -inf have probability 0.

    Returns (tokens int64 [..., K + 1], accepted int64 [...], log_probs [..., K + 1]): the accepted
    tokens, the drawn one and ignore_index behind it; how many were accepted; the target's
    log-probabilities of the tokens, 0 behind them (float32; float64 for float64 logits).  Where the
    target's logits hold NaN or +inf, or nothing but -inf, no token is drawn: ignore_index, with a
    log-probability of NaN.  Not differentiable.  The draw's sums are float64; the tests' are float32
    (float64 for float64 logits), so that a number within some 1e-7 of its border may go either way."""
    for t, name in ((logits, "logits"), (draft_tokens, "draft_tokens"), (uniforms, "uniforms")):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor")
    if not logits.is_cuda or draft_tokens.device != logits.device or uniforms.device != logits.device:
        raise RuntimeError("logits, draft_tokens and uniforms must be on the same HIP device")
    _dl.storage_dtype_code(logits)
    shape = logits.shape
    if len(shape) < 2 or shape[-2] < 1 or shape[-1] < 1:
        raise RuntimeError(f"logits must be [..., drafts + 1, classes], got shape {tuple(shape)}")
    lead, drafts = shape[:-2], shape[-2] - 1
    if draft_tokens.dtype != torch.int64 or draft_tokens.shape != (*lead, drafts):
        raise RuntimeError(f"draft_tokens must be int64 of shape {(*lead, drafts)}")
    if uniforms.dtype not in (torch.float32, torch.float64) or uniforms.shape != shape[:-1]:
        raise RuntimeError(f"uniforms must be float32 or float64 of shape {tuple(shape[:-1])}")
    if draft_logits is not None:
        if not isinstance(draft_logits, torch.Tensor):
            raise TypeError("draft_logits must be a tensor or None")
        if draft_logits.device != logits.device or draft_logits.dtype != logits.dtype \
                or draft_logits.shape != (*lead, drafts, shape[-1]):
            raise RuntimeError(f"draft_logits must be {logits.dtype} of shape "
                               f"{(*lead, drafts, shape[-1])} on {logits.device}")
        if drafts == 0:
            draft_logits = None
    if len(shape) != 3:
        count = lead.numel()
        logits = logits.reshape(count, drafts + 1, shape[-1])
        draft_tokens = draft_tokens.reshape(count, drafts)
        uniforms = uniforms.reshape(count, drafts + 1)
        if draft_logits is not None:
            draft_logits = draft_logits.reshape(count, drafts, shape[-1])
    tokens, accepted, log_probs = _native.load().verify_drafts(
        logits, draft_tokens.contiguous(), draft_logits, uniforms.contiguous(), int(ignore_index))
    if len(shape) != 3:
        return (tokens.reshape(shape[:-1]), accepted.reshape(lead), log_probs.reshape(shape[:-1]))
    return tokens, accepted, log_probs
