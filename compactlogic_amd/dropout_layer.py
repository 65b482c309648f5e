"""Dropout between logic layers on the HIP kernels (cl_dropout).  No counterpart in the reference.

The mask is not stored: it is a function of a seed, an offset and the element's place, Philox
4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC'11) with
the seed as its key and (column / 8, row, offset) as its counter, sixteen bits an element.  The
backward makes it again, a later evaluation of the same batch can ask for the same mask (a policy
and the one it is compared with), and it does not depend on how the tensor lies in memory.
"""
from __future__ import annotations

import torch

from . import _native
from . import difflogic_hip as _dl
from .layers import PackBitsTensor


def _threshold(p) -> int:
    if not 0 <= p <= 1:
        raise ValueError(f"dropout probability must be in [0, 1], got {p}")
    return int(round(65536 * float(p)))


def dropout(x, p: float, seed, offset: int = 0, fill: float | None = None):
    """Each element of x dropped with probability p, taken to the nearest multiple of 2^-16.

    fill=None: dropped elements become 0 and the others are divided by the probability of
    keeping them (the one that was taken), so that the mean stays; a number: dropped elements
    become that number and the others stay as they are (0.5, a bit that is not known, keeps a
    relaxed activation in [0, 1]).

    seed, offset: integers, or seed an int64 tensor (seed, offset) on x's device, read when the
    kernel runs (so a captured graph follows it).  Equal ones give equal masks: the first
    dimension is the row, the others together the column (so that Flatten may come before or
    after).  Where nothing can be dropped (p below 2^-17) x itself is returned."""
    if not isinstance(x, torch.Tensor):
        raise TypeError("x must be a tensor")
    if x.device.type != "cuda":
        raise RuntimeError("dropout needs a HIP device tensor")
    _dl.storage_dtype_code(x)
    threshold = _threshold(p)
    rng = None
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.shape != (2,) or seed.device != x.device:
            raise RuntimeError(f"seed must be an integer or an int64 tensor (seed, offset) on "
                               f"{x.device}")
        if offset != 0:
            raise ValueError("offset is part of a seed tensor")
        rng, seed = seed.contiguous(), 0
    if threshold == 0 or x.numel() == 0:
        return x
    flat = x if x.dim() == 2 else x.reshape(x.shape[0] if x.dim() > 2 else 1, -1)
    y = _native.load().dropout(flat, threshold, None if fill is None else float(fill),
                               int(seed) & (2**64 - 1), int(offset) & (2**64 - 1), rng)
    return y if x.dim() == 2 else y.reshape(x.shape)


class Dropout(torch.nn.Module):
    """`dropout` as a module, between the layers of a Sequential: in training every call draws the
    next mask (its buffer `rng` holds the seed and the count of calls, on the device, so a
    captured training step draws a new mask at every replay and a checkpoint resumes the
    sequence); in eval mode, and for a PackBitsTensor, the identity.  seed=None takes one from
    torch's generator.

    A segment that torch.utils.checkpoint runs again in the backward would draw another mask
    there, which is refused: take the mask before the segment and call the function in it,
    ``rng = drop.next_rng()`` and ``dropout(h, drop.p, rng, fill=drop.fill)``."""

    def __init__(self, p: float = 0.5, fill: float | None = None, seed: int | None = None):
        super().__init__()
        _threshold(p)
        self.p = p
        self.fill = fill
        if seed is None:
            seed = int(torch.randint(0, 2**63 - 1, (), device="cpu"))
        if not -2**63 <= seed < 2**63:
            raise ValueError("seed must fit in 64 bits")
        self.register_buffer("rng", torch.tensor([seed, 0], dtype=torch.int64))

    def next_rng(self) -> torch.Tensor:
        """The (seed, offset) of the next mask, as `dropout` takes it; advances the module."""
        if torch._C._current_graph_task_id() != -1:    # inside of a backward pass
            raise RuntimeError(
                "a Dropout module cannot draw its mask again in a backward pass, where "
                "torch.utils.checkpoint recomputes a segment: take rng = next_rng() before the "
                "segment and call dropout(x, p, rng, fill) in it")
        _dl._check(self.rng, "rng")
        return _native.load().dropout_next(self.rng)

    def forward(self, x):
        if not self.training or isinstance(x, PackBitsTensor) or _threshold(self.p) == 0:
            return x
        return dropout(x, self.p, self.next_rng(), fill=self.fill)

    def extra_repr(self):
        return f"p={self.p}, fill={self.fill}"
