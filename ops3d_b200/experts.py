"""Experts: which of them each token goes to, the rows sorted by expert in the form that ``grouped_linear`` takes, and back.

    weights, experts = route_experts(logits, top_k, bias=None, score="softmax", n_groups=1, top_groups=1, group_score="max",
                                     renormalise=True, scale=1.0)
        score = softmax(logits) or sigmoid(logits) ("softmax", "sigmoid"), select = score + bias
        experts: the ``top_k`` largest of select, largest first, among the experts of the ``top_groups`` best of ``n_groups`` equal runs of
        experts; a group is worth its largest select ("max") or the sum of its two largest ("top2")
        weights: ``scale * score / (sum of the chosen scores)``, without ``renormalise`` ``scale * score``
        logits ``[..., n_experts]``; bias ``[n_experts]`` float32; weights float32 and experts int64 ``[..., top_k]``

    rows, order = dispatch_rows(x, experts, n_experts)
        the row of x ``[..., features]`` for each entry of experts ``[..., top_k]``, sorted by expert, in the order of the entries
        within one; rows ``[tokens * top_k, features]``.  ``order.group_start_index`` ``[n_experts + 1]`` is what ``grouped_linear`` takes;
        ``order.position`` ``[..., top_k]`` is the row of each entry.  An entry outside ``0 .. n_experts - 1`` (a padded token's) belongs to
        no expert: its position is -1, and the rows behind the last expert's are 0.

    y = combine_rows(rows, order, weights=None, residual=None)
        the sum of ``weight * row`` over each token's entries, + residual; an entry of no expert adds nothing
        weights ``[..., top_k]`` (None: 1), residual and y ``[..., features]``

Ties go to the lower index.  Which experts are chosen does not depend on how an exponential rounds in fp32: scores that it cannot tell apart
are computed in 64 bits (which leaves sums of scores and biases that only differ beyond them).  Such tokens take longer: a peaked softmax or
saturated sigmoids beside a bias several times as long.  NaN compares as minus infinity and stays NaN in the weights; renormalised softmax weights
are the softmax over the chosen logits, and renormalised sigmoid weights are ratios that do not vanish where the scores do; a token whose scores
are all 0 (every logit minus infinity) has weights of 0.  The choice has no gradient: ``bias`` (kept
outside of training to balance the experts) gets none, logits get that of the weights.

CUDA tensors in float32, float16 or bfloat16 of any sizes and strides (one that is not contiguous is copied); index tensors int64.  Nothing is
read on the host, so everything may be captured into a graph.  Sums are fp32 in a fixed order, rounded once: repeated calls are
equal bit for bit.  Weights of ``combine_rows`` are float32 or in the dtype of the rows; a residual of another dtype than the rows' is
added behind the sum, in the wider of the two.  Up to 1024 experts, 32 entries a token, 32 groups, 2^31 - 1 entries.

``order`` comes from ``dispatch_rows``; entries may be taken out of it (``order._replace(position=...)`` with -1 for those beyond an
expert's capacity, say): their rows get a gradient of 0.  One put together by hand leads out of no tensor, but where entries share a row
its gradient is put together from theirs, not their sum.

``ExpertFeedForward`` is a transformer layer's feed-forward block with experts: norm, router, experts, sum and residual.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ._extension import _C, _C_IMPORT_ERROR
from .graph import takes_node
from .linear import FeedForward, add_residual, fused_linear, like
from .norm import LayerNorm

SCORES = {"softmax": 0, "sigmoid": 1}
GROUP_SCORES = {"max": 0, "top2": 1}


def _ext():
    if _C is None:
        raise RuntimeError(f"ops3d_b200._C extension not built; the operators of experts require it: {_C_IMPORT_ERROR}")
    return _C


def _code(codes: dict, name: str, value) -> int:
    try:
        return codes[value]
    except (KeyError, TypeError):
        raise ValueError(f"{name} must be one of {', '.join(codes)}; got {value!r}") from None


class RowOrder(NamedTuple):
    """Where ``dispatch_rows`` put each row."""

    group_start_index: torch.Tensor
    position: torch.Tensor


class RouteExpertsFunction(Function):
    """``apply(logits, bias, top_k, score, n_groups, top_groups, group_score, renormalise, scale)``, scores as codes.  ``apply`` is a C++
    graph node, ``forward`` and ``backward`` what it does where something has to see the Function itself (``graph.takes_node``)."""

    @staticmethod
    def forward(ctx, logits, bias, top_k, score, n_groups, top_groups, group_score, renormalise, scale):
        weights, experts = _ext().route_forward(logits, bias, top_k, score, n_groups, top_groups, group_score, renormalise, scale)
        ctx.options = (score, renormalise, scale)
        ctx.save_for_backward(logits, experts)
        ctx.mark_non_differentiable(experts)
        return weights, experts

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_weights, _):
        logits, experts = ctx.saved_tensors
        return (_ext().route_backward(logits, experts, grad_weights, *ctx.options), *[None] * 8)

    @classmethod
    def apply(cls, *args):
        if cls is RouteExpertsFunction and takes_node():
            return tuple(_ext().route(*args))
        return super().apply(*args)


def route_experts(logits, top_k, bias=None, score="softmax", n_groups=1, top_groups=1, group_score="max", renormalise=True, scale=1.0):
    """Weights and experts of each token (module docstring)."""
    return RouteExpertsFunction.apply(logits, bias, int(top_k), _code(SCORES, "score", score), int(n_groups), int(top_groups),
                                      _code(GROUP_SCORES, "group_score", group_score), bool(renormalise), float(scale))


class DispatchRowsFunction(Function):
    """``apply(x, experts, n_experts)`` -> ``(rows, group_start_index, position)``."""

    @staticmethod
    def forward(ctx, x, experts, n_experts):
        rows, starts, position = _ext().dispatch_forward(x, experts, n_experts)
        ctx.save_for_backward(position)
        ctx.mark_non_differentiable(starts, position)
        return rows, starts, position

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_rows, *_):
        (position,) = ctx.saved_tensors
        return _ext().combine_forward(grad_rows, position, None, None), None, None

    @classmethod
    def apply(cls, x, experts, n_experts):
        if cls is DispatchRowsFunction and takes_node():
            return tuple(_ext().dispatch(x, experts, n_experts))
        return super().apply(x, experts, n_experts)


def dispatch_rows(x, experts, n_experts):
    """The rows of x sorted by expert, and their order (module docstring)."""
    rows, starts, position = DispatchRowsFunction.apply(x, experts, int(n_experts))
    return rows, RowOrder(starts, position)


class CombineRowsFunction(Function):
    """``apply(rows, position, weights, residual)``."""

    @staticmethod
    def forward(ctx, rows, position, weights, residual):
        needs_rows = weights is not None and ctx.needs_input_grad[2]  # only the weights' gradient reads them
        ctx.save_for_backward(rows if needs_rows else None, position, weights)
        return _ext().combine_forward(rows, position, weights, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        need = ctx.needs_input_grad
        grad_rows, grad_weights = _ext().combine_backward(*ctx.saved_tensors, grad_output, need[0], need[2])
        return grad_rows, None, grad_weights, grad_output if need[3] else None

    @classmethod
    def apply(cls, rows, position, weights=None, residual=None):
        if cls is CombineRowsFunction and takes_node():
            return _ext().combine(rows, position, weights, residual)
        return super().apply(rows, position, weights, residual)


def combine_rows(rows, order, weights=None, residual=None):
    """Each token's weighted sum of its rows (module docstring)."""
    _, position = order
    if residual is None or residual.dtype == rows.dtype:
        return CombineRowsFunction.apply(rows, position, weights, residual)
    return add_residual(CombineRowsFunction.apply(rows, position, weights, None), residual)


class ExpertFeedForward(nn.Module):
    """``x + sum over a token's experts of weight * (W2 act(W1 h + b1) + b2)``, ``h = norm(x)`` (without the outer ``x`` where
    ``residual=False``, ``h = x`` where ``norm=False``).

    ``router`` ``[n_experts, d_model]`` makes the logits, in the rows' type (autocast's under autocast); the options are those of ``route_experts``.  With ``balanced`` a buffer
    ``balance`` is its bias: raise an expert's entry to send it more tokens.  ``forward`` takes a mask of tokens that are padding (True: no
    expert; it may hold anything) and with ``return_order`` returns the rows' order too, whose
    ``group_start_index.diff()`` is how many tokens each expert had."""

    def __init__(self, d_model: int = 256, d_hidden: int = 1024, n_experts: int = 8, top_k: int = 2, activation: str = "gelu",
                 score: str = "softmax", n_groups: int = 1, top_groups: int = 1, group_score: str = "max", renormalise: bool = True,
                 scale: float = 1.0, balanced: bool = False, norm: bool = True, residual: bool = True):
        super().__init__()
        _code(SCORES, "score", score)
        _code(GROUP_SCORES, "group_score", group_score)
        if n_groups < 1 or n_experts % n_groups or not 1 <= top_groups <= n_groups or not 1 <= top_k <= n_experts // n_groups * top_groups:
            raise ValueError("n_groups must divide n_experts, top_groups be in 1 .. n_groups and top_k fit the experts of top_groups groups")
        self.d_model, self.n_experts, self.top_k, self.residual = d_model, n_experts, top_k, residual
        self.routing = dict(score=score, n_groups=n_groups, top_groups=top_groups, group_score=group_score, renormalise=renormalise, scale=scale)
        self.norm = LayerNorm(d_model) if norm else None
        self.router = nn.Parameter(torch.empty(n_experts, d_model))
        nn.init.xavier_uniform_(self.router)
        if balanced:
            self.register_buffer("balance", torch.zeros(n_experts))
        else:
            self.balance = None
        self.experts = FeedForward(d_model, d_hidden, activation, n_groups=n_experts, residual=False)

    def forward(self, x, padding_mask=None, return_order=False):
        # nothing that padding holds, a NaN either, gets into the gradients of norm and router; no row of it is moved
        kept = x if padding_mask is None else x.masked_fill(padding_mask[..., None], 0.0)
        h = x if self.norm is None else self.norm(kept)
        balance = None if self.balance is None else self.balance.float()
        logits = fused_linear(kept if self.norm is None else h, like(h, self.router))
        weights, experts = route_experts(logits, self.top_k, balance, **self.routing)
        if padding_mask is not None:
            experts = experts.masked_fill(padding_mask[..., None], -1)
        rows, order = dispatch_rows(h, experts, self.n_experts)
        y = combine_rows(self.experts(rows, order.group_start_index), order, weights, x if self.residual else None)
        return (y, order) if return_order else y
