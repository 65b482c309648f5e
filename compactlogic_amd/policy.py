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

A small call spends most of its time in Python, on both sides of autograd: sizes are looked up
once per shape, what a call keeps to itself is one allocation, and there are few frames.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _capi
from . import difflogic_hip as _dl
from . import timing

_CODES = _dl._STORAGE_DTYPES
_F32, _F64 = torch.float32, torch.float64
_MEAN = _capi.CL_REDUCE["mean"]


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


def _rows_of(logits):
    """logits as the kernels read them: contiguous rows, any distance apart."""
    if logits.stride(1) != 1 and logits.shape[1] > 1:
        logits = logits.contiguous()
    return logits


# ---- sizes, once per shape

@functools.lru_cache(maxsize=4096)
def _prefills(code, rows, cols) -> bool:
    yes = ctypes.c_int()
    _capi.call("cl_policy_loss_prefills", code, rows, cols, ctypes.byref(yes))
    return bool(yes.value)


@functools.lru_cache(maxsize=4096)
def _centered_bytes(code, batch, feats, stride_batch, k) -> int:
    need = ctypes.c_int64()
    _capi.call("cl_group_sum_centered_workspace_size", code, batch, feats, stride_batch, k,
               ctypes.byref(need))
    return need.value


def takes_group(k: int) -> bool:
    """Whether the losses take GroupSum's scores of k classes from its input."""
    return _centered_bytes(_capi.CL_DTYPE_F32, 1, 1, 1, int(k)) >= 0


@functools.lru_cache(maxsize=4096)
def _buffer(code, rows, cols, *sizes):
    """The one buffer of a call: its bytes, the workspace's, and where the parts behind the rows'
    state start: those of `sizes` bytes, then the workspace; a multiple of 32 bytes each."""
    need = ctypes.c_int64()
    _capi.call("cl_token_loss_workspace", code, rows, cols, ctypes.byref(need))
    total, starts = 0, []
    for n in (4 * (8 if code == _capi.CL_DTYPE_F64 else 4) * rows, *sizes, need.value):
        starts.append(total)
        total += (n + 31) & ~31
    return max(total, 32), need.value, *starts[1:]


# ---- GroupSum's scores

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
    timing.launch(x, "cl_group_sum_centered_forward", code, x.data_ptr(), batch, feats, sb, sf, k,
                  tau, scores.data_ptr(), _dl.ptr(ws), need)
    ctx.group = k, tau, batch, feats, sb == 1 and sf != 1
    return scores


def _group_grad(ctx, scores, actions, at, row_grad=None, loss_grad=None, count=None, row_seq=None,
                seq_slope=None, pair_grad=None, pairs=0):
    """The gradient of GroupSum's input in its layout, formed from the scores where it is spread
    over the features."""
    k, tau, batch, feats, batch_major = ctx.group
    dtype, dev = scores.dtype, scores.device
    if batch_major:
        sb, sf = 1, batch
        grad_x = torch.empty_strided((batch, feats), (1, batch), dtype=dtype, device=dev)
    else:
        sb, sf = feats, 1
        grad_x = torch.empty((batch, feats), dtype=dtype, device=dev)
    timing.launch(scores, "cl_group_sum_chosen_backward", _CODES[dtype], scores.data_ptr(), batch,
                  feats, k, tau, actions.data_ptr(), at, row_grad, loss_grad, count, row_seq,
                  seq_slope, pair_grad, pairs, grad_x.data_ptr(), sb, sf)
    return grad_x


# ---- autograd

def _saved(ctx):
    """The logits, actions and buffer that a forward saved, wherever they lie now (hooks on saved
    tensors may have moved them).  The backwards are kernels without a derivative of their own:
    under create_graph a second derivative would silently lack its part."""
    if torch.is_grad_enabled():
        raise RuntimeError("the losses on chosen log-probabilities cannot be differentiated twice")
    logits, actions, aux = ctx.saved_tensors
    return _rows_of(logits), actions, aux


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
        dtype, dev = logits.dtype, logits.device
        code = _CODES[dtype]
        rows, cols = logits.shape
        total, ws_bytes, ws = _buffer(code, rows, cols)
        aux = torch.empty(total, dtype=torch.uint8, device=dev)
        lp = torch.empty(rows, dtype=_F64 if dtype == _F64 else _F32, device=dev)
        at = aux.data_ptr()
        timing.launch(logits, "cl_selected_log_prob_forward", code, logits.data_ptr(),
                      logits.stride(0), rows, cols, actions.data_ptr(), ignore_index,
                      lp.data_ptr(), at, at + ws, ws_bytes)
        ctx.save_for_backward(logits, actions, aux)   # (the rows' state comes first in aux)
        return lp

    @staticmethod
    def backward(ctx, grad_lp):
        logits, actions, aux = _saved(ctx)
        if not grad_lp.is_contiguous():
            grad_lp = grad_lp.contiguous()
        if ctx.group is not None:
            return _group_grad(ctx, logits, actions, aux.data_ptr(),
                               row_grad=grad_lp.data_ptr()), None, None, None
        rows, cols = logits.shape
        grad = torch.empty((rows, cols), dtype=logits.dtype, device=logits.device)
        timing.launch(logits, "cl_selected_log_prob_backward", _CODES[logits.dtype],
                      logits.data_ptr(), logits.stride(0), rows, cols, actions.data_ptr(),
                      aux.data_ptr(), grad_lp.data_ptr(), grad.data_ptr())
        return grad, None, None, None


class PolicyLossFunction(torch.autograd.Function):
    """The clipped policy loss with a KL term (cl_policy_loss_forward / _backward).  Returns (loss,
    log_probs); the log-probabilities are not differentiable through this function.  No
    counterpart in the reference."""

    @staticmethod
    def forward(ctx, x, actions, old, adv, ref, clip_low, clip_high, kl_coef, ignore_index,
                reduction, trains, group=None):
        logits = _logits_of(ctx, x, group)
        dtype, dev, wide = logits.dtype, logits.device, old.dtype
        code = _CODES[dtype]
        rows, cols = logits.shape
        size = 8 if dtype == _F64 else 4
        total, ws_bytes, count, terms, ws = _buffer(code, rows, cols, size,
                                                    size * rows if reduction else 0)
        aux = torch.empty(total, dtype=torch.uint8, device=dev)
        at = aux.data_ptr()
        lp = torch.empty(rows, dtype=wide, device=dev)
        loss = torch.empty(() if reduction else rows, dtype=wide, device=dev)
        loss_at = loss.data_ptr()
        grad = None
        if trains and reduction and group is None and _prefills(code, rows, cols):
            grad = torch.empty((rows, cols), dtype=dtype, device=dev)
            ctx.capture = _capture_id(logits)
        timing.launch(logits, "cl_policy_loss_forward", code, logits.data_ptr(), logits.stride(0),
                      rows, cols, actions.data_ptr(), ignore_index, old.data_ptr(),
                      adv.data_ptr(), None if ref is None else ref.data_ptr(), clip_low, clip_high,
                      kl_coef, reduction, lp.data_ptr(), at, at + terms if reduction else loss_at,
                      loss_at, at + count, None if grad is None else grad.data_ptr(), at + ws,
                      ws_bytes)
        ctx.save_for_backward(logits, actions, aux)
        ctx.grad, ctx.reduction, ctx.count = grad, reduction, count
        ctx.mark_non_differentiable(lp)
        ctx.set_materialize_grads(False)
        return loss, lp

    @staticmethod
    def backward(ctx, grad_loss, _grad_lp):
        if grad_loss is None:
            return (None,) * 12
        logits, actions, aux = _saved(ctx)
        if not grad_loss.is_contiguous():
            grad_loss = grad_loss.contiguous()
        reduction, at = ctx.reduction, aux.data_ptr()
        if ctx.group is not None:
            up = grad_loss.data_ptr()
            gx = _group_grad(ctx, logits, actions, at, loss_grad=up,
                             count=at + ctx.count if reduction == _MEAN else None) if reduction \
                else _group_grad(ctx, logits, actions, at, row_grad=up)
            return gx, None, None, None, None, None, None, None, None, None, None, None
        rows, cols = logits.shape
        # the forward's gradient is handed out once, and only in the capture (or outside of any)
        # that it was written in: a replay of the backward alone would find it used
        grad, ctx.grad = ctx.grad, None
        prefilled = grad is not None and ctx.capture == _capture_id(logits)
        if not prefilled:
            grad = torch.empty((rows, cols), dtype=logits.dtype, device=logits.device)
        timing.launch(logits, "cl_policy_loss_backward", _CODES[logits.dtype], logits.data_ptr(),
                      logits.stride(0), rows, cols, actions.data_ptr(), at, reduction,
                      grad_loss.data_ptr(), at + ctx.count, int(prefilled), grad.data_ptr())
        return grad, None, None, None, None, None, None, None, None, None, None, None


class PreferenceLossFunction(torch.autograd.Function):
    """The preference loss of paired sequences (cl_preference_loss_forward / _backward).  Returns
    (loss, margins); the margins are not differentiable through this function.  No counterpart in
    the reference."""

    @staticmethod
    def forward(ctx, x, actions, offsets, ref, beta, smoothing, ignore_index, reduction,
                group=None):
        logits = _logits_of(ctx, x, group)
        dtype, dev = logits.dtype, logits.device
        code = _CODES[dtype]
        rows, cols = logits.shape
        wide, size = (_F64, 8) if dtype == _F64 else (_F32, 4)
        pairs = (offsets.numel() - 1) // 2
        total, ws_bytes, count, row_seq, seq_slope, gaps, lp, terms, ws = _buffer(
            code, rows, cols, size, 4 * rows, 2 * pairs * size, 8 * rows, size * rows,
            size * pairs if reduction else 0)
        aux = torch.empty(total, dtype=torch.uint8, device=dev)
        at = aux.data_ptr()
        margins = torch.empty(pairs, dtype=wide, device=dev)
        loss = torch.empty(() if reduction else pairs, dtype=wide, device=dev)
        loss_at = loss.data_ptr()
        timing.launch(logits, "cl_preference_loss_forward", code, logits.data_ptr(),
                      logits.stride(0), rows, cols, actions.data_ptr(), ignore_index,
                      None if ref is None else ref.data_ptr(), offsets.data_ptr(), pairs, beta,
                      smoothing, reduction, at + lp, at, at + gaps, at + row_seq, at + seq_slope,
                      margins.data_ptr(), at + terms if reduction else loss_at, loss_at,
                      at + count, at + ws, ws_bytes)
        ctx.save_for_backward(logits, actions, aux)
        ctx.reduction, ctx.pairs, ctx.parts = reduction, pairs, (row_seq, seq_slope, count)
        ctx.mark_non_differentiable(margins)
        ctx.set_materialize_grads(False)
        return loss, margins

    @staticmethod
    def backward(ctx, grad_loss, _grad_margins):
        if grad_loss is None:
            return (None,) * 9
        logits, actions, aux = _saved(ctx)
        if not grad_loss.is_contiguous():
            grad_loss = grad_loss.contiguous()
        row_seq, seq_slope, count = ctx.parts
        at = aux.data_ptr()
        if ctx.group is not None:
            up, mean = grad_loss.data_ptr(), ctx.reduction == _MEAN
            gx = _group_grad(ctx, logits, actions, at, loss_grad=up if ctx.reduction else None,
                             count=at + count if mean else None, row_seq=at + row_seq,
                             seq_slope=at + seq_slope, pair_grad=None if ctx.reduction else up,
                             pairs=ctx.pairs)
            return gx, None, None, None, None, None, None, None, None
        rows, cols = logits.shape
        grad = torch.empty((rows, cols), dtype=logits.dtype, device=logits.device)
        timing.launch(logits, "cl_preference_loss_backward", _CODES[logits.dtype],
                      logits.data_ptr(), logits.stride(0), rows, cols, actions.data_ptr(), at,
                      at + row_seq, at + seq_slope, ctx.pairs, ctx.reduction,
                      grad_loss.data_ptr(), at + count, grad.data_ptr())
        return grad, None, None, None, None, None, None, None, None


# ---- public functions (_group: GroupSum's (k, tau), the logits then being its input)

def selected_log_probs(logits, actions, ignore_index: int = -100, *, _group=None):
    """The log-probability log_softmax(logits)[..., actions] of the chosen class or token:
    logits [..., V], actions int64 [...] -> [...]; 0 where the action is ignore_index.
    Differentiable by the logits."""
    rows, acts = _flat(logits, actions)
    lp = SelectedLogProbsFunction.apply(rows, acts, int(ignore_index), _group)
    return lp if actions.dim() == 1 else lp.reshape(actions.shape)


def policy_loss(logits, actions, old_log_probs, advantages, ref_log_probs=None, clip=0.2,
                kl_coef: float = 0.0, ignore_index: int = -100, reduction: str = "mean",
                return_log_probs: bool = False, *, _group=None):
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
    # (needs_input_grad is true under no_grad as well)
    trains = logits.requires_grad and torch.is_grad_enabled()
    loss, lp = PolicyLossFunction.apply(rows, acts, old, adv, ref, low, high, kl_coef,
                                        int(ignore_index), code, trains, _group)
    if actions.dim() != 1:
        lp = lp.reshape(actions.shape)
        if not code:
            loss = loss.reshape(actions.shape)
    return (loss, lp) if return_log_probs else loss


def preference_loss(logits, actions, offsets, ref_log_probs=None, beta: float = 0.1,
                    label_smoothing: float = 0.0, ignore_index: int = -100,
                    reduction: str = "mean", return_margins: bool = False, *, _group=None):
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
                                                 int(ignore_index), code, _group)
    return (loss, margins) if return_margins else loss
