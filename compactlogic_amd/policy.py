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
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _capi
from . import difflogic_hip as _dl
from . import timing


def _wide(logits: torch.Tensor) -> torch.dtype:
    return torch.float64 if logits.dtype == torch.float64 else torch.float32


def _flat(logits, actions):
    """logits (or the activations that GroupSum makes them of) as [rows, cols] and actions as
    [rows], checked."""
    if not isinstance(logits, torch.Tensor) or not isinstance(actions, torch.Tensor):
        raise TypeError("logits and actions must be tensors")
    if logits.device.type != "cuda" or actions.device != logits.device:
        raise RuntimeError("logits and actions must be on the same HIP device")
    _dl.storage_dtype_code(logits)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise RuntimeError(f"logits must have a last dimension of at least one class, got shape "
                           f"{tuple(logits.shape)}")
    if actions.dtype != torch.int64 or actions.shape != logits.shape[:-1]:
        raise RuntimeError(f"actions must be int64 of shape {tuple(logits.shape[:-1])}")
    if logits.dim() != 2:
        logits = logits.reshape(-1, logits.shape[-1])
        actions = actions.reshape(-1)
    return logits, actions.contiguous()


def _per_row(t, name, logits, actions):
    """A constant per row as a contiguous [rows] tensor of the logits' wide type."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.device != logits.device or t.shape != actions.shape or not t.is_floating_point():
        raise RuntimeError(f"{name} must be a floating-point tensor of shape "
                           f"{tuple(actions.shape)} on {logits.device}")
    if t.requires_grad:
        raise RuntimeError(f"{name} is a constant of the loss: detach it")
    wide = _wide(logits)
    if t.dim() != 1:
        t = t.reshape(-1)
    if t.dtype != wide:
        t = t.to(wide)
    return t if t.is_contiguous() else t.contiguous()


def _reduction(name):
    if name not in _capi.CL_REDUCE:
        raise ValueError(f"reduction must be one of {sorted(_capi.CL_REDUCE)}, got {name!r}")
    return _capi.CL_REDUCE[name]


def _rows_of(logits):
    """logits as the kernels read them: contiguous rows, any distance apart."""
    if logits.stride(1) != 1 and logits.shape[1] > 1:
        logits = logits.contiguous()
    return logits


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(code, rows, cols) -> int:
    need = ctypes.c_int64()
    _capi.call("cl_token_loss_workspace", code, rows, cols, ctypes.byref(need))
    return need.value


@functools.lru_cache(maxsize=1024)
def _prefills(code, rows, cols) -> bool:
    yes = ctypes.c_int()
    _capi.call("cl_policy_loss_prefills", code, rows, cols, ctypes.byref(yes))
    return bool(yes.value)


@functools.lru_cache(maxsize=1024)
def _centered_bytes(code, batch, feats, stride_batch, k) -> int:
    need = ctypes.c_int64()
    _capi.call("cl_group_sum_centered_workspace_size", code, batch, feats, stride_batch, k,
               ctypes.byref(need))
    return need.value


def takes_group(k: int) -> bool:
    """Whether the losses take GroupSum's scores of k classes from its input."""
    return _centered_bytes(_capi.CL_DTYPE_F32, 1, 1, 1, int(k)) >= 0


def _logits_of(ctx, x, group):
    """The rows of logits to work on: x itself, or, with group (k, tau), GroupSum's scores of the
    activations x [batch, features], less each sample's largest one (which no loss here depends
    on), so that they are not rounded at the size of a class sum."""
    ctx.group = None
    if group is None:
        return _rows_of(x)
    k, tau = group
    code = _dl.dtype_code(x)
    batch, feats = x.shape
    sb, sf = x.stride()
    if batch > 1 and feats > 1 and (sb == 0 or sf == 0):
        x = x.contiguous()
        sb, sf = x.stride()
    scores = torch.empty((batch, k), dtype=x.dtype, device=x.device)
    need = _centered_bytes(code, batch, feats, sb, k)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    with _dl.on_device_of(x):
        timing.call("cl_group_sum_centered_forward", code, x.data_ptr(), batch, feats, sb, sf, k,
                    tau, scores.data_ptr(), _dl.ptr(ws), need, _dl.stream_of(x))
    ctx.group = k, tau, batch, feats, sb == 1 and sf != 1
    return scores


def _input_grad(ctx, grad):
    """The input's gradient from the logits': through GroupSum, in its input's layout."""
    if ctx.group is None:
        return grad
    k, tau, batch, feats, batch_major = ctx.group
    if batch_major:
        grad_x = torch.empty((feats, batch), dtype=grad.dtype, device=grad.device).t()
    else:
        grad_x = torch.empty((batch, feats), dtype=grad.dtype, device=grad.device)
    sb, sf = grad_x.stride()
    with _dl.on_device_of(grad):
        timing.call("cl_group_sum_backward", _dl.dtype_code(grad), grad.data_ptr(), batch, feats,
                    k, tau, grad_x.data_ptr(), sb, sf, _dl.stream_of(grad))
    return grad_x


def _args(logits):
    """logits as the entry points take them (an expanded row has stride 0)."""
    rows, cols = logits.shape
    return _dl.storage_dtype_code(logits), logits.data_ptr(), logits.stride(0), rows, cols


class _Shape:
    """One call's logits as the entry points take them, and the bytes of its buffers."""

    def __init__(self, logits):
        self.args = code, _, _, rows, cols = _args(logits)
        self.code, self.rows, self.cols = code, rows, cols
        self.size = 8 if logits.dtype == torch.float64 else 4
        self.state_bytes = 4 * self.size * rows
        self.workspace_bytes = _workspace_bytes(code, rows, cols)


def _once():
    """The backwards are kernels without a derivative of their own: under create_graph a second
    derivative would silently lack its part."""
    if torch.is_grad_enabled():
        raise RuntimeError("the losses on chosen log-probabilities cannot be differentiated twice")


def _aux(logits, *sizes):
    """One buffer for everything a call keeps to itself, and where its parts start, a multiple of
    32 bytes each: allocations cost a small call more than its kernels."""
    total, starts = 0, []
    for n in sizes:
        starts.append(total)
        total += (n + 31) & ~31
    return torch.empty(max(total, 32), dtype=torch.uint8, device=logits.device), starts


def _saved(ctx):
    """The logits, actions and buffer that a forward saved, wherever they lie now (hooks on saved
    tensors may have moved them), and the logits as the entry points take them."""
    logits, actions, aux = ctx.saved_tensors
    logits = _rows_of(logits)
    return logits, actions, aux.data_ptr(), _args(logits), aux


def _capture_id(t) -> int:
    """Which graph capture t's current stream records, 0 outside of one."""
    got = ctypes.c_uint64()
    _capi.call("cl_stream_capture_id", _dl.stream_of(t), ctypes.byref(got))
    return got.value


class SelectedLogProbsFunction(torch.autograd.Function):
    """lp[n] = log_softmax(logits[n])[actions[n]] in one pass over the logits; the backward makes
    the probabilities again from the row's maximum and sum.  No counterpart in the reference."""

    @staticmethod
    def forward(ctx, x, actions, ignore_index, group=None):
        logits = _logits_of(ctx, x, group)
        sh = _Shape(logits)
        aux, (_, ws) = _aux(logits, sh.state_bytes, sh.workspace_bytes)
        at = aux.data_ptr()
        lp = torch.empty(sh.rows, dtype=_wide(logits), device=logits.device)
        with _dl.on_device_of(logits):
            timing.call("cl_selected_log_prob_forward", *sh.args, actions.data_ptr(), ignore_index,
                        lp.data_ptr(), at, at + ws, sh.workspace_bytes, _dl.stream_of(logits))
        ctx.save_for_backward(logits, actions, aux)   # (the rows' state comes first in aux)
        return lp

    @staticmethod
    def backward(ctx, grad_lp):
        _once()
        logits, actions, at, args, _kept = _saved(ctx)
        grad_lp = grad_lp.contiguous()
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        with _dl.on_device_of(logits):
            timing.call("cl_selected_log_prob_backward", *args, actions.data_ptr(), at,
                        grad_lp.data_ptr(), grad.data_ptr(), _dl.stream_of(logits))
        return _input_grad(ctx, grad), None, None, None


class PolicyLossFunction(torch.autograd.Function):
    """The clipped policy loss with a KL term (cl_policy_loss_forward / _backward).  Returns (loss,
    log_probs); the log-probabilities are not differentiable through this function.  No
    counterpart in the reference."""

    @staticmethod
    def forward(ctx, x, actions, old, adv, ref, clip_low, clip_high, kl_coef, ignore_index,
                reduction, group=None):
        logits = _logits_of(ctx, x, group)
        sh = _Shape(logits)
        wide = old.dtype
        lp = torch.empty(sh.rows, dtype=wide, device=logits.device)
        if reduction:
            loss = torch.empty((), dtype=wide, device=logits.device)
            aux, (_, ctx.count, terms, ws) = _aux(logits, sh.state_bytes, sh.size,
                                                  sh.rows * sh.size, sh.workspace_bytes)
            at = aux.data_ptr()
            terms, loss_at, count = at + terms, loss.data_ptr(), at + ctx.count
        else:
            loss = torch.empty(sh.rows, dtype=wide, device=logits.device)
            aux, (_, ws) = _aux(logits, sh.state_bytes, sh.workspace_bytes)
            at = aux.data_ptr()
            terms, loss_at, count = loss.data_ptr(), None, None
        grad = None
        if reduction and ctx.needs_input_grad[0] and _prefills(sh.code, sh.rows, sh.cols):
            grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
            ctx.capture = _capture_id(logits)
        with _dl.on_device_of(logits):
            timing.call("cl_policy_loss_forward", *sh.args, actions.data_ptr(), ignore_index,
                        old.data_ptr(), adv.data_ptr(), _dl.ptr(ref), clip_low, clip_high, kl_coef,
                        reduction, lp.data_ptr(), at, terms, loss_at, count, _dl.ptr(grad), at + ws,
                        sh.workspace_bytes, _dl.stream_of(logits))
        ctx.save_for_backward(logits, actions, aux)
        ctx.grad, ctx.reduction = grad, reduction
        ctx.mark_non_differentiable(lp)
        ctx.set_materialize_grads(False)
        return loss, lp

    @staticmethod
    def backward(ctx, grad_loss, _grad_lp):
        _once()
        if grad_loss is None:
            return (None,) * 11
        logits, actions, at, args, _kept = _saved(ctx)
        grad_loss = grad_loss.contiguous()
        # the forward's gradient is handed out once, and only in the capture (or outside of any)
        # that it was written in: a replay of the backward alone would find it used
        grad, ctx.grad = ctx.grad, None
        prefilled = grad is not None and ctx.capture == _capture_id(logits)
        if not prefilled:
            grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        with _dl.on_device_of(logits):
            timing.call("cl_policy_loss_backward", *args, actions.data_ptr(), at, ctx.reduction,
                        grad_loss.data_ptr(), at + ctx.count if ctx.reduction else None,
                        int(prefilled), grad.data_ptr(), _dl.stream_of(logits))
        return (_input_grad(ctx, grad),) + (None,) * 10


class PreferenceLossFunction(torch.autograd.Function):
    """The preference loss of paired sequences (cl_preference_loss_forward / _backward).  Returns
    (loss, margins); the margins are not differentiable through this function.  No counterpart in
    the reference."""

    @staticmethod
    def forward(ctx, x, actions, offsets, ref, beta, smoothing, ignore_index, reduction,
                group=None):
        logits = _logits_of(ctx, x, group)
        sh = _Shape(logits)
        wide, pairs = _wide(logits), (offsets.numel() - 1) // 2
        margins = torch.empty(pairs, dtype=wide, device=logits.device)
        loss = torch.empty(() if reduction else (pairs,), dtype=wide, device=logits.device)
        aux, (_, count, row_seq, seq_slope, gaps, lp, terms, ws) = _aux(
            logits, sh.state_bytes, sh.size, 4 * sh.rows, 2 * pairs * sh.size, 8 * sh.rows,
            sh.rows * sh.size, pairs * sh.size if reduction else 0, sh.workspace_bytes)
        at = aux.data_ptr()
        loss_at = loss.data_ptr() if reduction else None
        terms_at = at + terms if reduction else loss.data_ptr()
        with _dl.on_device_of(logits):
            timing.call("cl_preference_loss_forward", *sh.args, actions.data_ptr(), ignore_index,
                        _dl.ptr(ref), offsets.data_ptr(), pairs, beta, smoothing, reduction,
                        at + lp, at, at + gaps, at + row_seq, at + seq_slope, margins.data_ptr(),
                        terms_at, loss_at, at + count, at + ws, sh.workspace_bytes,
                        _dl.stream_of(logits))
        ctx.save_for_backward(logits, actions, aux)
        ctx.reduction, ctx.pairs, ctx.parts = reduction, pairs, (row_seq, seq_slope, count)
        ctx.mark_non_differentiable(margins)
        ctx.set_materialize_grads(False)
        return loss, margins

    @staticmethod
    def backward(ctx, grad_loss, _grad_margins):
        _once()
        if grad_loss is None:
            return (None,) * 9
        logits, actions, at, args, _kept = _saved(ctx)
        row_seq, seq_slope, count = ctx.parts
        grad_loss = grad_loss.contiguous()
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        with _dl.on_device_of(logits):
            timing.call("cl_preference_loss_backward", *args, actions.data_ptr(), at, at + row_seq,
                        at + seq_slope, ctx.pairs, ctx.reduction, grad_loss.data_ptr(), at + count,
                        grad.data_ptr(), _dl.stream_of(logits))
        return (_input_grad(ctx, grad),) + (None,) * 8


def selected_log_probs(logits, actions, ignore_index: int = -100):
    """The log-probability log_softmax(logits)[..., actions] of the chosen class or token:
    logits [..., V], actions int64 [...] -> [...]; 0 where the action is ignore_index.
    Differentiable by the logits."""
    return _selected_log_probs(logits, actions, ignore_index)


def _selected_log_probs(logits, actions, ignore_index=-100, group=None):
    rows, acts = _flat(logits, actions)
    lp = SelectedLogProbsFunction.apply(rows, acts, int(ignore_index), group)
    return lp if actions.dim() == 1 else lp.reshape(actions.shape)


def policy_loss(logits, actions, old_log_probs, advantages, ref_log_probs=None, clip=0.2,
                kl_coef: float = 0.0, ignore_index: int = -100, reduction: str = "mean",
                return_log_probs: bool = False):
    """The clipped policy loss with a KL term.  With lp the log-probability of the row's action,
    r = exp(lp - old_log_probs) and g = ref_log_probs - lp, a row's term is::

        -min(r A, clip(r, 1 - low, 1 + high) A) + kl_coef (exp(g) - g - 1)

    logits [..., V]; actions, old_log_probs (the acting policy's), advantages A and ref_log_probs
    (a frozen reference policy's, needed when kl_coef is not 0) [...].  clip: one number for both
    sides or a pair (low, high).  reduction: 'mean' over the rows that count, 'sum', or 'none' (the
    terms, [...]).  With return_log_probs, also the rows' log-probabilities (not differentiable
    through this call)."""
    return _policy_loss(logits, actions, old_log_probs, advantages, ref_log_probs, clip, kl_coef,
                        ignore_index, reduction, return_log_probs)


def _policy_loss(logits, actions, old_log_probs, advantages, ref_log_probs=None, clip=0.2,
                 kl_coef=0.0, ignore_index=-100, reduction="mean", return_log_probs=False,
                 group=None):
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
    loss, lp = PolicyLossFunction.apply(rows, acts, old, adv, ref, low, high, kl_coef,
                                        int(ignore_index), code, group)
    if actions.dim() != 1:
        lp = lp.reshape(actions.shape)
        if not code:
            loss = loss.reshape(actions.shape)
    return (loss, lp) if return_log_probs else loss


def preference_loss(logits, actions, offsets, ref_log_probs=None, beta: float = 0.1,
                    label_smoothing: float = 0.0, ignore_index: int = -100,
                    reduction: str = "mean", return_margins: bool = False):
    """The preference loss of P pairs of sequences out of one ragged batch.  Sequence q holds the
    rows offsets[q] .. offsets[q + 1] of logits [rows, V] and actions [rows] (offsets: int64
    [2 P + 1], not decreasing); the first P are the chosen sequences, sequence P + i is the one
    rejected against sequence i.  With D_q the sum of lp - ref_log_probs over a sequence's counted
    rows (ref_log_probs: a frozen reference policy's, [rows]; None: 0) and the margin
    h_i = beta (D_i - D_(P + i)), a pair's term is::

        -(1 - label_smoothing) log sigma(h) - label_smoothing log sigma(-h)

    reduction: 'mean' over the pairs, 'sum', or 'none' (the terms, [P]).  With return_margins, also
    the margins [P] (not differentiable through this call).  Rows of no sequence do not count;
    offsets that decrease or leave the rows make their pair's term NaN."""
    return _preference_loss(logits, actions, offsets, ref_log_probs, beta, label_smoothing,
                            ignore_index, reduction, return_margins)


def _preference_loss(logits, actions, offsets, ref_log_probs=None, beta=0.1, label_smoothing=0.0,
                     ignore_index=-100, reduction="mean", return_margins=False, group=None):
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
    loss, margins = PreferenceLossFunction.apply(rows, acts, offsets.contiguous(), ref,
                                                 float(beta), float(label_smoothing),
                                                 int(ignore_index), code, group)
    return (loss, margins) if return_margins else loss
