"""Fully connected product in 8-bit floating point and its gradients, with dropout folded in.

    y  = f q(m x) q(W)^T + b          blocks of 128 along the input features (weights: 128 x 128)
    dx = m f q(dy) q(W)               blocks along the output features
    dW = f q(dy^T) q((m x)^T)^T       blocks along the rows of the batch
    db = sum of dy over the batch

q(.) is the block quantiser of ``backend.ops.fp8_quantize_*``, m the 0/1 mask of ``backend.ops.dropout`` and f its factor
1 / (1 - p).  The mask is applied inside the quantiser and in the store of dx, the factor as the products' alpha: dropout
costs no pass over memory.  What the backward pass keeps is one byte per element of x and of W.
"""

from __future__ import annotations

import torch

from ..backend import _C


def linear_fp8(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, drop_p: float = 0.0,
               rng: torch.Tensor | None = None) -> torch.Tensor:
    """dropout(x) W^T + b with both operands of every product in block-scaled e4m3, forward and backward.

    x [..., in] fp32, bf16 or fp16 decides the result's type; weight [out, in] and bias [out] in any of these.  ``rng``
    (int64 {seed, offset}) is needed with ``drop_p`` > 0 and is read again in the backward pass.  There is no second derivative."""
    return _C.binding.linear_fp8(x, weight, bias, drop_p, rng)
