"""Layer norm with its backward pass, for rows in bf16 or fp32.

    y = layer_norm(x, weight, bias, eps)      differentiable in x, weight, bias
    LayerNorm(dim)                            the same as a module

The stock model normalises with RMSNorm (train.py:162-170), which
``SparseMoE.forward_normed`` folds into the layer; this is the norm of blocks that centre
their rows as well.  Statistics and the weight's and bias's gradients are fp32
whatever the rows' type, and the gradients have the same bits on every call.
"""

from __future__ import annotations

import torch
import torch.nn as nn
from torch.compiler import is_dynamo_compiling

from . import ops


def _param(p, rows, name):
    """An affine parameter as the kernels take it: (H,) contiguous fp32, beside the rows."""
    if p is None:
        return None
    if p.dim() != 1 or p.shape[0] != rows.shape[1]:
        raise RuntimeError(f"layer_norm: {name} must have shape ({rows.shape[1]},), got "
                           f"{tuple(p.shape)}")
    if p.get_device() != rows.get_device():
        raise RuntimeError(f"layer_norm: {name} must be a CUDA tensor on {rows.device} (no CPU "
                           "path)")
    if p.dtype is torch.float32 and p.is_contiguous():
        return p
    return p.detach().float().contiguous()


def _of_type(g, dtype, wanted):
    if not wanted:
        return None
    return g if g.dtype is dtype else g.to(dtype)


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        rows = ops.aligned_rows(ops.as_rows(x, "layer_norm"))
        w = _param(weight, rows, "weight")
        y, stats = ops.layer_norm_fwd(rows, w, _param(bias, rows, "bias"), eps, True, x)
        ctx.save_for_backward(rows, w, stats)
        ctx.types = tuple(None if p is None else p.dtype for p in (weight, bias))
        return y

    @staticmethod
    def backward(ctx, dy):
        ops.refuse_second_order("layer_norm")
        rows, w, stats = ctx.saved_tensors
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        g = ops.aligned_rows(ops.as_rows(dy, "layer_norm gradient"))
        dx, dw, db = ops.layer_norm_bwd(g, rows, w, stats, need_x, need_w or need_b, dy)
        wt, bt = ctx.types
        return dx, _of_type(dw, wt, need_w), _of_type(db, bt, need_b), None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension.

    x: bf16 or fp32 CUDA, any leading dimensions and row stride; weight and bias: of the last
    dimension's size, or None.  The result has x's type and shape."""
    if is_dynamo_compiling():
        return _outside_graph(x, weight, bias, eps)
    if ops.records(x, weight, bias):
        return _LayerNormFn.apply(x, weight, bias, eps)
    rows = ops.aligned_rows(ops.as_rows(x, "layer_norm"))
    y, _ = ops.layer_norm_fwd(rows, _param(weight, rows, "weight"), _param(bias, rows, "bias"), eps,
                              False, x)
    return y


_outside_graph = ops.outside_graph(layer_norm)


class LayerNorm(nn.Module):
    """``layer_norm`` with fp32 parameters, over the last dimension."""

    def __init__(self, dim: int, eps: float = 1e-5, bias: bool = True):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))
        self.bias = nn.Parameter(torch.zeros(dim)) if bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)
