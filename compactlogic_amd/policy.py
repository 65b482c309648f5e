"""Training by preference and by reward on the HIP kernels: losses on the log-probability of one
chosen class or token per row of logits, such as GroupSum's scores.

The reference trains classifiers with torch's cross_entropy alone; these have no counterpart
there.  `selected_log_probs` records what a policy (the acting one, or a frozen reference) gives
to the chosen actions, `policy_loss` and `preference_loss` train on them; GroupSum has all three
as methods, beside its cross_entropy.  Logits may be float32, float64, float16 or bfloat16; sums
and softmax statistics are float32 or more, and log-probabilities, losses and what they are
computed from are float32 (float64 for float64 logits).

A row whose action is ``ignore_index`` (a prompt or padding) does not count: its log-probability
and its gradient are 0 whatever its other inputs hold, NaN included.  Another action outside the
logits' range gives NaN, as a label does in GroupSum.cross_entropy.

The autograd Functions are C++ (csrc/autograd.cpp): a small call spends its time on the host, on both
sides of autograd.  Arguments are checked here.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _capi, _native
from . import difflogic_hip as _dl

_CODES = _dl._STORAGE_DTYPES
_F32, _F64 = torch.float32, torch.float64
_NO_GROUP = 0, 1.0


def _flat(logits, actions):
    """logits (or the activations that GroupSum makes them of) as [rows, cols] and actions as
    [rows], checked."""
    if not isinstance(logits, torch.Tensor) or not isinstance(actions, torch.Tensor):
        raise TypeError("logits and actions must be tensors")
    if not logits.is_cuda or actions.device != logits.device:
        raise RuntimeError("logits and actions must be on the same HIP device")
    if logits.dtype not in _CODES:
        _dl.storage_dtype_code(logits)
    shape = logits.shape
    if not shape or shape[-1] < 1:
        raise RuntimeError(f"logits must have a last dimension of at least one class, got shape "
                           f"{tuple(shape)}")
    if actions.dtype != torch.int64 or actions.shape != shape[:-1]:
        raise RuntimeError(f"actions must be int64 of shape {tuple(shape[:-1])}")
    if len(shape) != 2:
        logits = logits.reshape(-1, shape[-1])
        actions = actions.reshape(-1)
    return logits, actions if actions.is_contiguous() else actions.contiguous()


def _per_row(t, name, like, actions):
    """A constant per row as a contiguous [rows] tensor of the type that goes with `like`."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.device != like.device or t.shape != actions.shape or not t.is_floating_point():
        raise RuntimeError(f"{name} must be a floating-point tensor of shape "
                           f"{tuple(actions.shape)} on {like.device}")
    if t.requires_grad:
        raise RuntimeError(f"{name} is a constant of the loss: detach it")
    wide = _F64 if like.dtype == _F64 else _F32
    if t.dim() != 1:
        t = t.reshape(-1)
    if t.dtype != wide:
        t = t.to(wide)
    return t if t.is_contiguous() else t.contiguous()


def _reduction(name):
    code = _capi.CL_REDUCE.get(name)
    if code is None:
        raise ValueError(f"reduction must be one of {sorted(_capi.CL_REDUCE)}, got {name!r}")
    return code


@functools.lru_cache(maxsize=4096)
def _prefills(code, rows, cols) -> bool:
    """Whether the policy loss takes the logits' gradient along with the loss."""
    yes = ctypes.c_int()
    _capi.call("cl_policy_loss_prefills", code, rows, cols, ctypes.byref(yes))
    return bool(yes.value)


@functools.lru_cache(maxsize=64)
def takes_group(k: int) -> bool:
    """Whether the losses take GroupSum's scores of k classes from its input."""
    need = ctypes.c_int64()
    _capi.call("cl_group_sum_centered_workspace_size", _capi.CL_DTYPE_F32, 1, 1, 1, int(k),
               ctypes.byref(need))
    return need.value >= 0


# ---- public functions (_group: GroupSum's k and tau, the logits then being its input)

def selected_log_probs(logits, actions, ignore_index: int = -100, *, _group=_NO_GROUP):
    """The log-probability log_softmax(logits)[..., actions] of the chosen class or token:
    logits [..., V], actions int64 [...] -> [...]; 0 where the action is ignore_index.
    Differentiable by the logits."""
    rows, acts = _flat(logits, actions)
    lp = _native.load().selected_log_probs(rows, acts, int(ignore_index), *_group)
    return lp if actions.dim() == 1 else lp.reshape(actions.shape)


def policy_loss(logits, actions, old_log_probs, advantages, ref_log_probs=None, clip=0.2,
                kl_coef: float = 0.0, ignore_index: int = -100, reduction: str = "mean",
                return_log_probs: bool = False, *, _group=_NO_GROUP):
    """The clipped policy loss with a KL term.  With lp the log-probability of the row's action,
    r = exp(lp - old_log_probs) and g = ref_log_probs - lp, a row's term is::

        -min(r A, clip(r, 1 - low, 1 + high) A) + kl_coef (exp(g) - g - 1)

    logits [..., V]; actions, old_log_probs (the acting policy's), advantages A and ref_log_probs
    (a frozen reference policy's, needed when kl_coef is not 0) [...].  clip: one number for both
    sides or a pair (low, high).  reduction: 'mean' over the rows that count, 'sum', or 'none' (the
    terms, [...]).  With return_log_probs, also the rows' log-probabilities (not differentiable
    through this call).

    Large float32 and bfloat16 logits get their gradient along with a scalar loss, as it is for
    loss.backward().  A scaled loss (divided by a number of accumulated batches) forms it again;
    scaling advantages and kl_coef instead, in which the loss is linear, saves that."""
    rows, acts = _flat(logits, actions)
    low, high = (clip, clip) if isinstance(clip, (int, float)) else clip
    low, high, kl_coef = float(low), float(high), float(kl_coef)
    if not (low >= 0 and high >= 0):
        raise ValueError(f"clip must not be negative, got {clip}")
    if kl_coef != 0 and ref_log_probs is None:
        raise ValueError("a KL term (kl_coef) needs ref_log_probs")
    code = _reduction(reduction)
    old = _per_row(old_log_probs, "old_log_probs", logits, actions)
    adv = _per_row(advantages, "advantages", logits, actions)
    ref = None
    if ref_log_probs is not None:
        ref = _per_row(ref_log_probs, "ref_log_probs", logits, actions)
    prefill = code and _group is _NO_GROUP and logits.requires_grad and torch.is_grad_enabled() \
        and _prefills(_CODES[logits.dtype], *rows.shape)
    loss, lp = _native.load().policy_loss(rows, acts, old, adv, ref, low, high, kl_coef,
                                          int(ignore_index), code, bool(prefill), *_group)
    if actions.dim() != 1:
        lp = lp.reshape(actions.shape)
        if not code:
            loss = loss.reshape(actions.shape)
    return (loss, lp) if return_log_probs else loss


def preference_loss(logits, actions, offsets, ref_log_probs=None, beta: float = 0.1,
                    label_smoothing: float = 0.0, ignore_index: int = -100,
                    reduction: str = "mean", return_margins: bool = False, *, _group=_NO_GROUP):
    """The preference loss of P pairs of sequences out of one ragged batch.  Sequence q holds the
    rows offsets[q] .. offsets[q + 1] of logits [rows, V] and actions [rows] (offsets: int64
    [2 P + 1], not decreasing); the first P are the chosen sequences, sequence P + i is the one
    rejected against sequence i.  With D_q the sum of lp - ref_log_probs over a sequence's counted
    rows (ref_log_probs: a frozen reference policy's, [rows]; None: 0) and the margin
    h_i = beta (D_i - D_(P + i)), a pair's term is::

        -(1 - label_smoothing) log sigma(h) - label_smoothing log sigma(-h)

    reduction: 'mean' over the pairs, 'sum', or 'none' (the terms, [P]).  With return_margins, also
    the margins [P] (not differentiable through this call).  Rows of no sequence do not count;
    offsets that decrease or leave the rows make their pair's term NaN, and a decrease the gradient
    of the rows inside of it, which may lie in several sequences."""
    rows, acts = _flat(logits, actions)
    if logits.dim() != 2:
        raise RuntimeError("preference_loss takes logits [rows, classes] of a ragged batch")
    if not isinstance(offsets, torch.Tensor):
        raise TypeError("offsets must be a tensor")
    if offsets.device != logits.device or offsets.dtype != torch.int64 or offsets.dim() != 1 \
            or offsets.numel() % 2 != 1:
        raise RuntimeError(f"offsets must be int64 [2 pairs + 1] on {logits.device}")
    if not 0 <= label_smoothing <= 1:
        raise ValueError(f"label_smoothing must be in [0, 1], got {label_smoothing}")
    code = _reduction(reduction)
    ref = None
    if ref_log_probs is not None:
        ref = _per_row(ref_log_probs, "ref_log_probs", logits, actions)
    loss, margins = _native.load().preference_loss(rows, acts, offsets.contiguous(), ref,
                                                   float(beta), float(label_smoothing),
                                                   int(ignore_index), code, *_group)
    return (loss, margins) if return_margins else loss
