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
from torch.autograd import Function

from ..backend import ops as _ops

_F8 = torch.float8_e4m3fn


def _rows(x):
    return x.reshape(-1, x.shape[-1])


class _linear_fp8(Function):

    @staticmethod
    def forward(ctx, x, weight, bias, drop_p, rng):
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        alpha = _ops.drop_factor(drop_p)
        x2 = _rows(x)
        xt = xts = wt = wts = None
        if need_w:
            xq, xs, xt, xts = _ops.fp8_quantize_both(x2, _F8, drop_p, rng)
        else:
            xq, xs = _ops.fp8_quantize_rows(x2, _F8, drop_p, rng)
        if need_x:
            wq, ws, wt, wts = _ops.fp8_quantize_blocks(weight, _F8)
        else:
            wq, ws = _ops.fp8_quantize_blocks(weight, _F8, transposed=False)
        y = _ops.fp8_gemm(xq, xs, wq, ws, bias, alpha, x.dtype)
        ctx.save_for_backward(xt, xts, wt, wts, rng if _ops.drop_threshold(drop_p) else None)
        ctx.drop_p, ctx.alpha, ctx.x_shape, ctx.x_dtype = drop_p, alpha, x.shape, x.dtype
        ctx.w_dtype, ctx.b_dtype = weight.dtype, None if bias is None else bias.dtype
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    def backward(ctx, grad_output):
        xt, xts, wt, wts, rng = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        go = _rows(grad_output)
        dx = dw = db = None
        if need_w:
            gq, gs, gt, gts = _ops.fp8_quantize_both(go, _F8)
            dw = _ops.fp8_gemm(gt, gts, xt, xts, None, ctx.alpha, ctx.w_dtype)
        elif need_x:
            gq, gs = _ops.fp8_quantize_rows(go, _F8)
        if need_x:
            dx = _ops.fp8_gemm(gq, gs, wt, wts, None, ctx.alpha, ctx.x_dtype, ctx.drop_p, rng).view(ctx.x_shape)
        if need_b:
            db = go.sum(0, dtype=torch.float32).to(ctx.b_dtype)
        return dx, dw, db, None, None


def linear_fp8(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, drop_p: float = 0.0,
               rng: torch.Tensor | None = None) -> torch.Tensor:
    """dropout(x) W^T + b with both operands of every product in block-scaled e4m3, forward and backward.

    x [..., in] fp32, bf16 or fp16 decides the result's type; weight [out, in] and bias [out] in any of these.  ``rng``
    (int64 {seed, offset}) is needed with ``drop_p`` > 0 and is read again in the backward pass."""
    if x.dim() == 0 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise RuntimeError(f"expected x [..., {tuple(weight.shape)[-1:]}] and weight [out, in], got {tuple(x.shape)} and {tuple(weight.shape)}")
    return _linear_fp8.apply(x, weight, bias, drop_p, rng)
