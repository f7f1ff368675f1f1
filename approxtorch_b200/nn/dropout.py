"""Dropout whose mask is drawn from a counter-based generator and never stored.

The reference has no dropout of its own; its models use torch's, which keeps a mask (or a generator's state) for the
backward pass.  Here element i is kept or not by (seed, offset, i) alone, so the backward pass draws the same mask again,
and ``gemm_fp8.linear_fp8`` applies it inside its quantiser and its gradient product without a pass of its own.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from ..backend import _C, ops as _ops


def counter_dropout(x: torch.Tensor, p: float, rng: torch.Tensor) -> torch.Tensor:
    """x / (1 - p) where kept, 0 elsewhere, with gradient.  ``rng``: int64 {seed, offset} on x's device; it is read again in
    the backward pass, so pass a state that stays as it is (``backend.ops.dropout_advance`` hands one out)."""
    return _C.binding.counter_dropout(x, p, rng)


def new_state(seed: int | None) -> torch.Tensor:
    """{seed, 0}; without a seed, one from torch's default generator."""
    if seed is None:
        seed = int(torch.randint(2 ** 62, ()))
    return torch.tensor([seed, 0], dtype=torch.int64)


class CounterDropout(nn.Module):
    """Dropout layer on ``counter_dropout``.  Its state {seed, offset} is a buffer: it moves on by one on the device with
    every training forward (also in replays of a captured graph), is saved in checkpoints, and decides the masks, so a
    resumed run draws what the interrupted one would have drawn.  Give every rank its own seed, and wrap the model with
    ``broadcast_buffers=False`` (DistributedDataParallel otherwise hands rank 0's state to all).

    A forward that is run again for the backward pass (``torch.utils.checkpoint``) has to draw what it drew the first time:
    take the state before, ``rng = backend.ops.dropout_advance(layer.rng)``, and hand it to ``layer(x, rng)``.  Without it
    the second run draws anew, and the gradient is that of another mask."""

    def __init__(self, p: float = 0.5, seed: int | None = None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout probability must be between 0 and 1, got {p}")
        self.p = p
        self.register_buffer('rng', new_state(seed))

    def forward(self, x: torch.Tensor, rng: torch.Tensor | None = None) -> torch.Tensor:
        if not self.training or self.p == 0.0:
            return x
        return counter_dropout(x, self.p, _ops.dropout_advance(self.rng) if rng is None else rng)

    def extra_repr(self) -> str:
        return f"p={self.p}"
