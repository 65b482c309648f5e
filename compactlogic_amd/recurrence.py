"""Recurrences over sequences of logic activations on the HIP kernels.  No counterpart in the
reference.

A relaxed multiplexer whose output is fed back, ``h = g h + (1 - g) x``, is the relaxation of a
latch: on binary gates and inputs it holds (1) or takes its input (0) exactly.  As the recurrence is
linear in h, a long sequence need not be walked step by step: the steps of a stretch of time are one
linear map, and maps are joined in any grouping (csrc/recurrence.hip).
"""
from __future__ import annotations

import torch

from . import _native
from .layers import LogicLayer, PackBitsTensor, to_rows

_FORMS = {"mix": 0, "add": 1}


def gated_recurrence(x, gate, state=None, form: str = "mix", return_state: bool = False):
    """``h_t = g_t h_(t-1) + (1 - g_t) x_t`` (form "mix") or ``h_t = g_t h_(t-1) + x_t`` ("add")
    over the time of x and gate [batch, time, features] from state [batch, features] (None: 0).
    Returns h [batch, time, features] in x's type, and with return_state also the last state
    [batch, features] in float32 (float64), from which a later call goes on: one step at a time
    gives what the whole sequence gives, up to rounding, while the state is handed on as it is.

    x and gate: float32, float64, float16 or bfloat16.  Features or times may lie contiguous (a
    LogicLayer's output for batch * time samples has its times so, and the result lies alike); other
    layouts are copied.  States and arithmetic are float32 (float64), each result is rounded once.
    Differentiable once by x, gate and state, through the outputs and the last state; not in forward
    mode, whose tangents are refused.

    A gate of exactly 0 drops what came before, and one of exactly 1 leaves x unread in "mix": a
    sequence may begin anew inside of a row, or end before it, whatever the other steps hold, NaN
    included (the gate's own gradient is the formula's there).  Gates may be of any magnitude, also where
    a run of them multiplies past the largest number over states that are 0 or small.  Stretches of time
    with such runs are walked, which takes longer (where times are contiguous, from gates on whose
    product over 4 float32 or 8 16-bit steps is above 16)."""
    code = _FORMS.get(form)
    if code is None:
        raise ValueError(f"form must be one of {sorted(_FORMS)}, got {form!r}")
    y, last = _native.load().gated_recurrence(x, gate, state, code)   # (the tensors are checked there)
    return (y, last) if return_state else y


class LogicRecurrence(torch.nn.Module):
    """A layer of latches: one LogicLayer computes each latch's gate from the step's input, one its
    data, and a latch holds where its gate is 1 and takes its data where it is 0.

    x [batch, time, in_dim] -> [batch, time, out_dim], from a state [batch, out_dim] (None: zeros);
    with return_state also the state behind the last step, for the next call.  In eval mode, or
    frozen, gates and data are the discrete ones of `LogicLayer`, and so is the result for binary
    inputs.  Packed inputs are not supported.  The other arguments are LogicLayer's."""

    def __init__(self, in_dim: int, out_dim: int, connections: str = 'random', num_gates=16,
                 residual_init: bool = False):
        super().__init__()
        self.in_dim = in_dim
        self.out_dim = out_dim
        self.gate = LogicLayer(in_dim, out_dim, connections, num_gates, residual_init)
        self.data = LogicLayer(in_dim, out_dim, connections, num_gates, residual_init)

    def forward(self, x, state=None, return_state: bool = False):
        if isinstance(x, PackBitsTensor):
            raise RuntimeError("LogicRecurrence takes sequences of activations, not packed bits")
        if x.dim() != 3 or x.shape[2] != self.in_dim:
            raise RuntimeError(f"x must be [batch, time, {self.in_dim}], got {tuple(x.shape)}")
        steps = x.shape[:2]
        if steps.numel() == 0:
            empty = x.new_zeros((*steps, self.out_dim))
            return gated_recurrence(empty, empty, state, return_state=return_state)
        rows = to_rows(x.reshape(-1, self.in_dim)).transpose(0, 1)
        gate, data = self.gate(rows), self.data(rows)
        return gated_recurrence(data.unflatten(0, steps), gate.unflatten(0, steps), state,
                                return_state=return_state)

    def freeze(self):
        self.gate.freeze()
        self.data.freeze()

    def extra_repr(self):
        return f"{self.in_dim}, {self.out_dim}"
