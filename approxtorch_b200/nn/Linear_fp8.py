"""Fully connected layer on the block-scaled 8-bit floating point product: the native low-precision counterpart of
``Linear_int8`` (which looks every product up in a table), for layers that are not simulated and as the yardstick for
those that are.  Master weights stay in their own type; every forward quantises them anew unless they are frozen.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn

from ..backend import ops as _ops
from .dropout import new_state
from .gemm_fp8 import linear_fp8


class Linear_fp8(nn.Module):
    """y = dropout(x) W^T + b.  ``dropout`` is applied in training only, its state {seed, offset} is the buffer ``rng`` (see
    ``CounterDropout``, also for forwards that are run twice); ``state_dict`` keys of ``weight`` and ``bias`` are those of
    ``nn.Linear``.

    A training step can be captured into a CUDA graph.  Let go of every result that was computed from the same parameters on
    the default stream first (warm up on a side stream): while one lives, a captured backward pass raises RuntimeError."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, dropout: float = 0.0, seed: int | None = None):
        super().__init__()
        if not 0.0 <= dropout <= 1.0:
            raise ValueError(f"dropout probability must be between 0 and 1, got {dropout}")
        self.in_features, self.out_features, self.dropout = in_features, out_features, dropout
        self.weight = nn.Parameter(torch.empty(out_features, in_features))
        self.bias = nn.Parameter(torch.empty(out_features)) if bias else None
        if dropout > 0.0:
            self.register_buffer('rng', new_state(seed))
        self._frozen = None
        nn.init.kaiming_uniform_(self.weight, a=math.sqrt(5))      # nn.Linear's default
        if self.bias is not None:
            bound = 1 / math.sqrt(in_features) if in_features > 0 else 0
            nn.init.uniform_(self.bias, -bound, bound)

    def freeze_weight(self):
        """Quantise the weights once for the forwards that want no gradient (serving).  Later changes of ``weight`` are
        not seen until ``unfreeze_weight`` or another ``freeze_weight``; moving the layer or loading a checkpoint unfreezes."""
        self._frozen = _ops.fp8_quantize_blocks(self.weight.detach(), transposed=False)

    def unfreeze_weight(self):
        self._frozen = None

    def _apply(self, fn, recurse=True):
        self._frozen = None
        return super()._apply(fn, recurse)

    def _load_from_state_dict(self, *args, **kwargs):
        self._frozen = None
        return super()._load_from_state_dict(*args, **kwargs)

    def forward(self, x: torch.Tensor, rng: torch.Tensor | None = None) -> torch.Tensor:
        if x.dim() == 0 or x.shape[-1] != self.in_features:
            raise RuntimeError(f"expected last dimension {self.in_features}, got {tuple(x.shape)}")
        p = self.dropout if self.training else 0.0
        if p > 0.0 and rng is None:
            rng = _ops.dropout_advance(self.rng)
        wants_grad = torch.is_grad_enabled() and (
            x.requires_grad or self.weight.requires_grad or (self.bias is not None and self.bias.requires_grad))
        if self._frozen is not None and not wants_grad:
            xq, xs = _ops.fp8_quantize_rows(x.reshape(-1, self.in_features), drop_p=p, rng=rng)
            y = _ops.fp8_gemm(xq, xs, *self._frozen, self.bias, _ops.drop_factor(p), x.dtype)
            return y.view(*x.shape[:-1], self.out_features)
        return linear_fp8(x, self.weight, self.bias, p, rng)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, dropout={self.dropout}"
