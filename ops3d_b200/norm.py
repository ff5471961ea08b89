"""Layer norm of a residual sum, forward and backward, in one pass over memory each.

    layer_norm(x, weight=None, bias=None, residual=None, eps=1e-5, return_sum=False)
        s = x + residual,   y = (s - mean(s)) / sqrt(var(s) + eps) * weight + bias      over the last dimension
        x, y ``[..., features]``, weight, bias ``[features]``, residual ``[..., features]``
        ``return_sum``: ``(y, s)``, for a stream that goes on behind the norm

CUDA tensors of any sizes and strides (one that is not contiguous is copied); x in float32, float16 or bfloat16 and y like it; weight and
bias in the dtype of x or float32, both the same; the residual, and s with it, in the dtype of x or float32 (a stream that keeps its bits around a
16-bit layer).  Sums, statistics and s as y sees it are fp32; every output is rounded once.  Gradients reach x, weight, bias and
residual, once.  Nothing but the inputs is kept for the backward, which takes the statistics from them again.  Parameter gradients are
summed in a fixed order: repeated calls are equal bit for bit.  Up to 2^31 - 1 rows and 2^26 - 1 features.  A NaN or an infinity
makes its own row NaN (and, in the backward, the parameters' gradients).

Autocast changes nothing: the statistics are fp32 anyway, and y has the dtype of x.

``LayerNorm`` holds weight and bias; its state dict is that of ``torch.nn.LayerNorm`` over the last dimension.
"""
from __future__ import annotations

import torch
from torch import nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ._extension import _C, _C_IMPORT_ERROR
from .graph import takes_node


def _ext():
    if _C is None:
        raise RuntimeError(f"ops3d_b200._C extension not built; layer_norm requires it: {_C_IMPORT_ERROR}")
    return _C


class LayerNormFunction(Function):
    """``apply(x, weight, bias, residual, eps, return_sum)`` -> ``(y, s)``, s None without ``return_sum``.  ``apply`` is a C++ graph node,
    ``forward`` and ``backward`` what it does where something has to see the Function itself (``graph.takes_node``)."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps, return_sum):
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, residual)
        y, s = _ext().layer_norm_forward(x, weight, bias, residual, eps, return_sum)
        return y, s

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y, grad_sum):
        x, weight, bias, residual = ctx.saved_tensors
        if grad_y is None:
            grad_y = torch.zeros_like(x)
        grads = _ext().layer_norm_backward(x, weight, bias, residual, grad_y, grad_sum, ctx.eps, *ctx.needs_input_grad[:4])
        return (*grads, None, None)

    @classmethod
    def apply(cls, x, weight=None, bias=None, residual=None, eps=1e-5, return_sum=False):
        if cls is LayerNormFunction and takes_node():
            return tuple(_ext().layer_norm(x, weight, bias, residual, eps, return_sum))
        return super().apply(x, weight, bias, residual, eps, return_sum)


def layer_norm(x, weight=None, bias=None, residual=None, eps=1e-5, return_sum=False):
    """Layer norm of ``x + residual`` over the last dimension (module docstring)."""
    if return_sum and residual is None:
        raise ValueError("return_sum needs a residual; without one the sum is x")
    y, s = LayerNormFunction.apply(x, weight, bias, residual, float(eps), bool(return_sum))
    return (y, s) if return_sum else y


class LayerNorm(nn.Module):
    """``layer_norm`` with its parameters, which stay fp32 beside 16-bit rows."""

    def __init__(self, features: int, eps: float = 1e-5, bias: bool = True):
        super().__init__()
        self.features, self.eps = features, eps
        self.weight = nn.Parameter(torch.ones(features))
        self.bias = nn.Parameter(torch.zeros(features)) if bias else None

    def forward(self, x, residual=None, return_sum=False):
        return layer_norm(x, self.weight, self.bias, residual, self.eps, return_sum)
