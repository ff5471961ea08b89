"""Linear layers with everything around the product in one pass, and the same with one weight per ragged group of rows.

    fused_linear(x, weight, bias=None, residual=None, activation="none")
        y = act(x @ weight^T + bias) + residual
        x ``[..., in]``, weight ``[out, in]``, bias ``[out]``, residual and y ``[..., out]``

    grouped_linear(x, weight, group_start_index, bias=None, residual=None, activation="none")
        the same with ``weight[e]``, ``bias[e]`` for the rows of group e
        x ``[rows, in]`` or ``[batch, rows, in]``, weight ``[groups, out, in]``, bias ``[groups, out]``

``group_start_index`` is an int64 CUDA tensor like the operator's ``level_start_index``: group e holds the rows from its entry to the
next one's of every batch element; the last group ends with the rows, or at one more entry where there is one.  Nothing is read
on the host, so the groups may change inside a captured graph.  An index below an earlier one counts as that one, indices
outside ``0 .. rows`` as the nearer end; an empty group is fine.  Rows of no group have no product: ``y = residual`` or 0 there.

Activations: ``"none"``, ``"relu"``, ``"gelu"`` (``v Phi(v)``), ``"gelu_tanh"``, ``"silu"``.  All tensors are CUDA tensors of one dtype --
float32, float16 or bfloat16 -- of any sizes and strides (an operand that is not contiguous is copied).  Sums are kept in
fp32 and rounded once.  Nothing but the inputs is kept for the backward, which computes ``x @ weight^T + bias`` again where
the activation's derivative needs it; beyond 64 rows ``grad_output * act'`` is rounded to the inputs' dtype between the backward's
products (not in the sums for the bias).  The results of repeated calls are equal bit for bit.  Up to 1024 groups, 2^31 - 1 rows and 2^26 - 1 features.
``gelu`` is 0 at minus infinity.

Under ``torch.autocast("cuda")`` x, weight and bias are taken in autocast's dtype, as torch's own linear layers take them.  A residual of
another dtype (an fp32 stream) is then added behind the product, and the result has the wider of the two.

Blocks of the 16-bit kernels wait for one another, two seconds at most (never in a sound run): results that a wait ran out on are NaN, and
``linear_timeouts()`` counts it.

``FeedForward`` is a transformer layer's ``x + W2 act(W1 x + b1) + b2``, with a weight pair of its own per group of rows where
``n_groups`` is given (one per pyramid level, or one per expert).
"""
from __future__ import annotations

import torch
from torch import nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ._extension import _C, _C_IMPORT_ERROR
from .graph import takes_node

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def _ext():
    if _C is None:
        raise RuntimeError(f"ops3d_b200._C extension not built; the linear operators require it: {_C_IMPORT_ERROR}")
    return _C


def _activation_code(activation: str) -> int:
    try:
        return ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}; got {activation!r}") from None


class FusedLinearFunction(Function):
    """``apply(x, weight, bias, residual, group_start_index, activation)``; ``group_start_index`` None: one weight for all rows.
    Gradients reach x, weight, bias and residual, once.  ``apply`` is a C++ graph node, ``forward`` and ``backward`` what it does
    where something has to see the Function itself (``graph.takes_node``)."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, group_start_index, activation):
        ctx.code = _activation_code(activation)
        ctx.save_for_backward(x, weight, bias, group_start_index)
        return _ext().linear_forward(x, weight, bias, residual, group_start_index, ctx.code)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        x, weight, bias, starts = ctx.saved_tensors
        need = ctx.needs_input_grad
        grads = (None, None, None)
        if any(need[:3]):
            grads = _ext().linear_backward(x, weight, bias, starts, grad_output, ctx.code, *need[:3])
        return (*grads, grad_output if need[3] else None, None, None)

    @classmethod
    def apply(cls, x, weight, bias=None, residual=None, group_start_index=None, activation="none"):
        if cls is FusedLinearFunction and takes_node():
            return _ext().linear(x, weight, bias, residual, group_start_index, _activation_code(activation))
        return super().apply(x, weight, bias, residual, group_start_index, activation)


def _product(x, weight, bias, residual, group_start_index, activation):
    """``FusedLinearFunction.apply``, under autocast with x, weight and bias in its dtype (float64 stays, and is refused) and a residual of
    another dtype added behind the product."""
    if not torch.is_autocast_enabled("cuda"):
        return FusedLinearFunction.apply(x, weight, bias, residual, group_start_index, activation)
    dtype = torch.get_autocast_dtype("cuda")
    x, weight, bias = (t if t is None or t.dtype in (dtype, torch.float64) or not t.is_floating_point() else t.to(dtype) for t in (x, weight, bias))
    if residual is None or residual.dtype == x.dtype:
        return FusedLinearFunction.apply(x, weight, bias, residual, group_start_index, activation)
    return add_residual(FusedLinearFunction.apply(x, weight, bias, None, group_start_index, activation), residual)


def fused_linear(x, weight, bias=None, residual=None, activation="none"):
    """``act(x @ weight^T + bias) + residual`` in one pass (module docstring)."""
    return _product(x, weight, bias, residual, None, activation)


def grouped_linear(x, weight, group_start_index, bias=None, residual=None, activation="none"):
    """``fused_linear`` with a weight per group of rows (module docstring)."""
    if group_start_index is None:
        raise ValueError("group_start_index is required; fused_linear takes one weight for all rows")
    return _product(x, weight, bias, residual, group_start_index, activation)


def linear_timeouts() -> int:
    """How many waits inside the operators' kernels have run out on the current device: 0 in a sound process.  Synchronises with the device."""
    return _ext().linear_timeouts()


def like(x, parameter):
    """``parameter`` in the dtype of ``x`` (a 16-bit input beside fp32 parameters); under autocast itself, for the call to cast it once."""
    if parameter is None or parameter.dtype == x.dtype or torch.is_autocast_enabled("cuda"):
        return parameter
    return parameter.to(x.dtype)


def add_residual(y, residual):
    """``y + residual`` in the wider of their dtypes, for a residual that the product's epilogue does not take."""
    if residual.shape != y.shape:
        raise RuntimeError(f"residual must have the shape of the output, {list(y.shape)}, got {list(residual.shape)}")
    return y + residual


class GroupedLinear(nn.Module):
    """``grouped_linear`` with its parameters: ``n_groups`` linear layers, each for its own rows."""

    def __init__(self, n_groups: int, in_features: int, out_features: int, bias: bool = True, activation: str = "none"):
        super().__init__()
        _activation_code(activation)
        self.n_groups, self.in_features, self.out_features, self.activation = n_groups, in_features, out_features, activation
        self.weight = nn.Parameter(torch.empty(n_groups, out_features, in_features))
        self.bias = nn.Parameter(torch.empty(n_groups, out_features)) if bias else None
        self._reset_parameters()

    def _reset_parameters(self):
        for each in self.weight:
            nn.init.xavier_uniform_(each)
        if self.bias is not None:
            nn.init.constant_(self.bias, 0.0)

    def forward(self, x, group_start_index, residual=None):
        return grouped_linear(x, like(x, self.weight), group_start_index, like(x, self.bias), residual, self.activation)


class FeedForward(nn.Module):
    """``x + W2 act(W1 x + b1) + b2`` (without the outer ``x`` where ``residual=False``): two calls of the operators above.

    ``n_groups``: a weight pair per group of rows; ``forward`` then takes their ``group_start_index`` (an encoder's
    ``level_start_index`` for one pair per pyramid level, or where each expert's rows begin in rows sorted by expert)."""

    def __init__(self, d_model: int = 256, d_hidden: int = 1024, activation: str = "relu", n_groups: int | None = None, residual: bool = True):
        super().__init__()
        _activation_code(activation)
        self.d_model, self.d_hidden, self.activation, self.n_groups, self.residual = d_model, d_hidden, activation, n_groups, residual
        lead = () if n_groups is None else (n_groups,)
        self.weight1 = nn.Parameter(torch.empty(*lead, d_hidden, d_model))
        self.bias1 = nn.Parameter(torch.empty(*lead, d_hidden))
        self.weight2 = nn.Parameter(torch.empty(*lead, d_model, d_hidden))
        self.bias2 = nn.Parameter(torch.empty(*lead, d_model))
        self._reset_parameters()

    def _reset_parameters(self):
        for w, b in ((self.weight1, self.bias1), (self.weight2, self.bias2)):
            for each in (w if w.dim() == 3 else w[None]):
                nn.init.xavier_uniform_(each)
            nn.init.constant_(b, 0.0)

    def forward(self, x, group_start_index=None):
        if (self.n_groups is None) != (group_start_index is None):
            raise ValueError("group_start_index goes with n_groups")
        w1, b1, w2, b2 = (like(x, p) for p in (self.weight1, self.bias1, self.weight2, self.bias2))
        hidden = _product(x, w1, b1, None, group_start_index, self.activation)
        return _product(hidden, w2, b2, x if self.residual else None, group_start_index, "none")
