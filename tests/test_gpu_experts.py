"""Routing to experts, rows sorted by expert and back, against the definitions in 64 bits.

Choices, positions and start indices have to be equal.  Tolerances of numbers, with u = 2^-24 (half a step of fp32):

* a softmax score is off by u (|l - max| + 4) from its exponential, by as much in the mean over the row and 40 u more from the sum, 3 u from the
  quotient; a sigmoid score by 7 u; a renormalised weight by twice the largest of its scores' errors and 12 u
* gradients of logits: their terms' magnitudes times three times that and 20 u
* a sum of n products in fp32: (n + 2) u of the sum of their magnitudes
* a rounding to the output's type: half a step
"""
import itertools
import math
import threading

import pytest
import torch

from ops3d_b200 import (CombineRowsFunction, DispatchRowsFunction, ExpertFeedForward, RouteExpertsFunction, combine_rows, dispatch_rows,
                        grouped_linear, linear_timeouts, route_experts)

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24
INF, NAN = float("inf"), float("nan")


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    assert linear_timeouts() == 0


def rounding(v, dtype):
    fi = torch.finfo(dtype)
    return v.abs() * (fi.eps / 2) * (1 + fi.eps) * 1.02 + fi.tiny * fi.eps / 2


def close(got, value, bound, name=""):
    value, bound = value.reshape(got.shape), bound.reshape(got.shape) + rounding(value, got.dtype).reshape(got.shape)
    assert torch.isfinite(got).all(), name
    worst = ((got.detach().double() - value).abs() / bound.clamp_min(1e-300)).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3f} of the bound"


# ---- routing ------------------------------------------------------------------------------------------------------------------
def chosen(logits, k, bias=None, score="softmax", n_groups=1, top_groups=1, group_score="max", **_):
    """The experts in 64 bits; scores of which one is a function of one logit are compared by the logits."""
    l = logits.double()
    s = torch.softmax(l, -1) if score == "softmax" else torch.sigmoid(l)
    s = torch.where((l == -INF).all(-1, keepdim=True), torch.zeros_like(s), s)
    v = l if bias is None else s + bias.double()
    v = torch.where(v.isnan(), -INF, v) + 0.0
    if top_groups < n_groups:
        each = (v if group_score == "max" or logits.shape[-1] == n_groups else s if bias is None else v).unflatten(-1, (n_groups, -1))
        each = each.sort(-1, descending=True).values
        worth = each[..., 0] if group_score == "max" or each.shape[-1] == 1 else each[..., 0] + each[..., 1]
        worth = torch.where(worth.isnan(), -INF, worth)
        best = worth.sort(dim=-1, descending=True, stable=True).indices[..., :top_groups]
        keep = torch.zeros_like(worth, dtype=torch.bool).scatter_(-1, best, True).repeat_interleave(each.shape[-1], -1)
    else:
        keep = torch.ones_like(v, dtype=torch.bool)
    # candidates first, then by value: a candidate of minus infinity comes before any other expert
    order = v.sort(dim=-1, descending=True, stable=True).indices
    first = keep.gather(-1, order).to(torch.int8).sort(dim=-1, descending=True, stable=True).indices
    return order.gather(-1, first)[..., :k]


def weights_of(logits, experts, score="softmax", renormalise=True, scale=1.0, dw=None, **_):
    """Weights and the logits' gradient with their bounds."""
    l = logits.double()
    e = l.shape[-1]
    if score == "softmax":
        top = l.max(-1, keepdim=True).values
        p = torch.softmax(l, -1)
        far = torch.where(l == -INF, 0.0, (l - top).abs())
        rel = U * (far + 4 + (p * (far + 4)).sum(-1, keepdim=True) + 43)
    else:
        p = torch.sigmoid(l)
        rel = torch.full_like(l, 7 * U)
    c, cr = p.gather(-1, experts), rel.gather(-1, experts)
    if renormalise:
        total = c.sum(-1, keepdim=True)
        w = scale * c / total
        wr = 2 * cr.max(-1, keepdim=True).values + 12 * U
        if score == "softmax":  # from the chosen logits alone
            lc = l.gather(-1, experts)
            wr = 2 * U * ((lc.max(-1, keepdim=True).values - lc) + 8).max(-1, keepdim=True).values + 12 * U
    else:
        total, w, wr = torch.ones_like(c[..., :1]), scale * c, cr + 2 * U
    out = dict(weights=(w, w * wr))
    if dw is None:
        return out
    dw = dw.double() * scale
    if renormalise:
        ds = (dw - (dw * c).sum(-1, keepdim=True) / total) / total
        mag = (dw.abs() + (dw.abs() * c).sum(-1, keepdim=True) / total) / total
    else:
        ds, mag = dw, dw.abs()
    if score == "sigmoid":
        grad = torch.zeros_like(l).scatter(-1, experts, ds * c * (1 - c))
        # 1 - s is off by what s is off by
        bound = torch.zeros_like(l).scatter(-1, experts, mag * c * ((1 - c) * (3 * wr + 20 * U) + 8 * U * c))
    else:
        along, amag = (ds * c).sum(-1, keepdim=True), (mag * c).sum(-1, keepdim=True)
        grad = torch.zeros_like(l).scatter(-1, experts, ds * c) - p * along
        dense = torch.zeros_like(l) if renormalise else p * amag * (3 * rel + 3 * wr.max(-1, keepdim=True).values + 20 * U)
        if renormalise:
            grad = torch.zeros_like(l).scatter(-1, experts, grad.gather(-1, experts))     # a softmax over the chosen
        bound = dense.scatter_add(-1, experts, (mag + amag) * c * (3 * wr + 20 * U))
    out["grad"] = (grad, bound)
    return out


def check_route(logits, k, bias=None, seed=0, **options):
    leaf = logits.detach().requires_grad_(True)
    weights, experts = route_experts(leaf, k, bias=bias, **options)
    assert weights.dtype == F32 and experts.dtype == torch.int64 and weights.shape == experts.shape == (*logits.shape[:-1], k)
    want = chosen(logits, k, bias, **options)
    assert torch.equal(experts, want), (experts != want).any(-1).sum()
    dw = torch.randn(weights.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))
    ref = weights_of(logits, experts, dw=dw, **options)
    close(weights, *ref["weights"], "weights")
    (grad,) = torch.autograd.grad(weights, leaf, dw)
    assert grad.dtype == logits.dtype and grad.shape == logits.shape
    close(grad, *ref["grad"], "grad_logits")


def logits_of(tokens, experts, dtype=F32, seed=0, scale=1.5):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(tokens, experts, generator=gen, device=DEV) * scale).to(dtype)


EXPERTS = [1, 2, 5, 24, 31, 32, 33, 63, 64, 65, 100, 128, 129, 200, 256, 257, 333, 512, 513, 777, 1024]


@pytest.mark.parametrize("experts", EXPERTS)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_choices(experts, score):
    for i, (dtype, biased, renormalise) in enumerate(itertools.product((F32, F16, BF16), (False, True), (False, True))):
        k = [1, 2, 3, 6, 8, 16, 32][(i + experts) % 7]
        bias = torch.randn(experts, device=DEV, generator=torch.Generator(device=DEV).manual_seed(i)) * 0.05 if biased else None
        check_route(logits_of(41, experts, dtype, seed=experts + i), min(k, experts), bias, score=score, renormalise=renormalise, scale=1.0 + i % 2)


@pytest.mark.parametrize("experts,groups", [(8, 2), (24, 3), (64, 8), (60, 4), (65, 13), (96, 32), (200, 8), (256, 8), (510, 2), (1024, 32), (32, 32),
                                            (1020, 5)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_choices_within_groups(experts, groups, score):
    for i, (dtype, biased, group_score) in enumerate(itertools.product((F32, BF16), (False, True), ("max", "top2"))):
        top_groups = 1 + (experts + i) % groups
        k = min(1 + (3 * i) % 9, top_groups * (experts // groups), 32)
        bias = torch.randn(experts, device=DEV, generator=torch.Generator(device=DEV).manual_seed(i)) * 0.05 if biased else None
        check_route(logits_of(37, experts, dtype, seed=experts + i), k, bias, score=score, n_groups=groups, top_groups=top_groups, group_score=group_score,
                    renormalise=i % 2 == 0)


def test_many_tokens_and_shapes():
    check_route(logits_of(40001, 64, BF16), 6, torch.zeros(64, device=DEV), score="sigmoid", n_groups=8, top_groups=3, group_score="top2")
    check_route(logits_of(30001, 24), 2)
    check_route(logits_of(24, 40).view(2, 3, 4, 40), 3)
    check_route(logits_of(1, 40)[0], 3)
    weights, experts = route_experts(torch.zeros(0, 8, device=DEV), 2)
    assert weights.shape == experts.shape == (0, 2)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides(dtype):
    wide = logits_of(50, 80, dtype)
    for view in (wide.t(), wide[:, ::2], wide[:, 1:], wide[:1].expand(9, 80)):
        check_route(view, 4, torch.linspace(-0.1, 0.1, 2 * view.shape[-1], device=DEV)[::2])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts", [24, 64, 300])
def test_ties_go_to_the_lower_index(experts, score):
    """Few distinct logits, with and without a bias of few distinct values: most choices are among equals."""
    logits = (logits_of(200, experts) * 1.0).round().clamp(-2, 2)
    levels = (torch.arange(experts, device=DEV) % 3).float() * 0.25
    for bias in (None, torch.zeros(experts, device=DEV), levels):
        for groups, top in ((1, 1), (4, 2)):
            for group_score in ("max", "top2"):
                check_route(logits, 6, bias, score=score, n_groups=groups, top_groups=top, group_score=group_score)
    same = torch.zeros(3, experts, device=DEV)
    assert torch.equal(route_experts(same, 5, score=score)[1], torch.arange(5, device=DEV).expand(3, 5))
    signed = torch.where(torch.arange(experts, device=DEV) % 2 == 0, -0.0, 0.0).expand(3, experts).contiguous()
    assert torch.equal(route_experts(signed, 5, score=score)[1], torch.arange(5, device=DEV).expand(3, 5))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups", [(64, 1), (200, 1), (64, 8)])
def test_values_that_fp32_cannot_tell_apart(experts, groups, score):
    """A bias that takes every token's score away: what is left are differences of a part in 2^26 and less."""
    row = logits_of(1, experts, seed=5)
    s = torch.softmax(row.double(), -1) if score == "softmax" else torch.sigmoid(row.double())
    bias = (0.7 - s[0]).float()
    near = row + torch.linspace(-2e-6, 2e-6, 64, device=DEV)[:, None] * torch.randn(64, experts, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    left = (torch.sigmoid(near.double()) if score == "sigmoid" else torch.softmax(near.double(), -1)) + bias.double()
    gaps = left.sort(-1).values.diff(dim=-1)
    assert (gaps > 0).all() and gaps.median() < 2.0 ** -26       # distinct in 64 bits, hardly any in 32
    for group_score in ("max", "top2"):
        options = dict(score=score, n_groups=groups, top_groups=(groups + 1) // 2, group_score=group_score)
        assert torch.equal(route_experts(near, 8, bias=bias, **options)[1], chosen(near, 8, bias, **options))


def test_masked_experts():
    """Minus infinity and the types' lowest value as masks; rows of which nothing is left."""
    for dtype in (F32, F16, BF16):
        logits = logits_of(64, 40, dtype)
        mask = torch.rand(64, 40, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3)) < 0.5
        for value in (-INF, torch.finfo(dtype).min):
            masked = logits.masked_fill(mask, value)
            for renormalise in (True, False):
                check_route(masked, 4, renormalise=renormalise)
                check_route(masked, 4, torch.zeros(40, device=DEV), score="sigmoid", renormalise=renormalise)
        off = torch.where(torch.arange(40, device=DEV) % 2 == 0, -INF, 0.0)
        check_route(logits, 4, off)                                         # a bias that switches experts off
        assert (route_experts(logits, 20, bias=off)[1] % 2 == 1).all()
        nothing = torch.full((3, 40), -INF, dtype=dtype, device=DEV, requires_grad=True)
        for score, renormalise, bias in itertools.product(("softmax", "sigmoid"), (True, False), (None, torch.zeros(40, device=DEV))):
            weights, experts = route_experts(nothing, 4, bias=bias, score=score, renormalise=renormalise)
            assert not weights.any() and torch.equal(experts, torch.arange(4, device=DEV).expand(3, 4))
            (grad,) = torch.autograd.grad(weights, nothing, torch.ones_like(weights))
            assert not grad.any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("experts", [24, 64, 128, 256, 512, 1000])
def test_rows_of_one_value(dtype, experts):
    """Every logit the same, the types' extremes among them: the first experts, equal weights, and no gradient through a softmax of all."""
    fi = torch.finfo(dtype)
    for value in (0.0, -3.0, fi.min, fi.max, fi.tiny):
        logits = torch.full((5, experts), value, dtype=dtype, device=DEV)
        for bias in (None, torch.full((experts,), 0.25, device=DEV)):
            for renormalise in (True, False):
                weights, chosen_ = route_experts(logits, 4, bias=bias, renormalise=renormalise)
                assert torch.equal(chosen_, torch.arange(4, device=DEV).expand(5, 4))
                assert (weights - 1 / (4 if renormalise else experts)).abs().max() <= 60 * U / (4 if renormalise else experts)
            weights, chosen_ = route_experts(logits, 4, bias=bias, score="sigmoid", renormalise=False)
            want = torch.sigmoid(torch.tensor(value, dtype=torch.float64)).item()
            assert torch.equal(chosen_, torch.arange(4, device=DEV).expand(5, 4)) and (weights - want).abs().max() <= 8 * U * want + 2.0 ** -148


def test_choices_of_less_than_all_that_is_left():
    """Two experts are left of which four are wanted: the others follow by index, with weights of 0."""
    logits = torch.full((2, 10), -INF, device=DEV)
    logits[0, 7], logits[0, 3] = 1.0, 2.0
    logits[1, 9] = 0.0
    weights, experts = route_experts(logits, 4)
    assert experts.tolist() == [[3, 7, 0, 1], [9, 0, 1, 2]]
    assert not weights[0, 2:].any() and weights[1].tolist() == [1.0, 0.0, 0.0, 0.0]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_nan_and_infinity(score, biased):
    """Indices stay distinct and in range, other tokens keep their results, NaN is not hidden."""
    logits = logits_of(8, 40)
    bias = torch.zeros(40, device=DEV) if biased else None
    good = route_experts(logits, 4, bias=bias, score=score, renormalise=False)
    bad = logits.clone()
    bad[1, 5], bad[3], bad[5, 6], bad[5, 7] = NAN, NAN, INF, INF
    for groups in (1, 4):
        for group_score in ("max", "top2"):
            weights, experts = route_experts(bad, 4, bias=bias, score=score, renormalise=False, n_groups=groups, top_groups=(groups + 1) // 2,
                                             group_score=group_score)
            assert ((experts >= 0) & (experts < 40)).all()
            assert all(len(set(row)) == 4 for row in experts.tolist())
            if groups == 1:
                assert torch.equal(experts[[0, 2, 4, 6, 7]], good[1][[0, 2, 4, 6, 7]]) and torch.equal(weights[[0, 2, 4, 6, 7]], good[0][[0, 2, 4, 6, 7]])
            assert weights[3].isnan().all()
            if score == "softmax":
                assert weights[1].isnan().all()


def test_route_gradient_against_differences():
    logits = logits_of(7, 20).requires_grad_(True)
    for score, renormalise in itertools.product(("softmax", "sigmoid"), (True, False)):
        weights, experts = route_experts(logits, 3, score=score, renormalise=renormalise, scale=2.5)
        dw = torch.randn(7, 3, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0))
        (grad,) = torch.autograd.grad(weights, logits, dw)
        v = torch.randn(7, 20, dtype=torch.float64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))

        def quotient(h):
            a, b = ((weights_of(logits.detach().double() + t * v, experts, score, renormalise, 2.5)["weights"][0] * dw).sum() for t in (h, -h))
            return ((a - b) / (2 * h)).item()

        near, far = quotient(2.0 ** -12), quotient(2.0 ** -11)
        value, bound = weights_of(logits.detach(), experts, score, renormalise, 2.5, dw)["grad"]
        slack = ((bound + rounding(value, F32)) * v.abs()).sum().item()
        assert abs((grad.double() * v).sum().item() - near) <= slack + abs(near - far) + 1e-9 * abs(near)


# ---- rows ---------------------------------------------------------------------------------------------------------------------
def order_of(experts, n_experts):
    """The definition, on the host."""
    flat = experts.reshape(-1).cpu()
    position = torch.full_like(flat, -1)
    starts = [0]
    for e in range(n_experts):
        mine = (flat == e).nonzero()[:, 0]
        position[mine] = starts[-1] + torch.arange(mine.numel())
        starts.append(starts[-1] + mine.numel())
    return torch.tensor(starts).to(DEV), position.view(experts.shape).to(DEV)


def rows_of(shape, dtype, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def check_rows(experts, n_experts, width, dtype, weights="f32", residual=True, seed=0):
    lead, k = experts.shape[:-1], experts.shape[-1]
    n = experts.numel()
    starts, position = order_of(experts, n_experts)
    flat = position.reshape(-1)
    there = flat >= 0
    at = flat.clamp_min(0)
    x = rows_of((*lead, width), dtype, seed).requires_grad_(True)
    rows, order = dispatch_rows(x, experts, n_experts)
    assert torch.equal(order.group_start_index, starts) and torch.equal(order.position, position)
    want = torch.zeros(n, width, dtype=dtype, device=DEV)
    want[flat[there]] = x.detach().reshape(-1, 1, width).expand(-1, k, width).reshape(n, width)[there]
    assert rows.shape == (n, width) and torch.equal(rows, want)
    dr = rows_of((n, width), dtype, seed + 1)
    (gx,) = torch.autograd.grad(rows, x, dr)
    each = (dr.double()[at] * there[:, None]).view(-1, k, width) if n else dr.double().view(-1, k, width)
    close(gx, each.sum(1), (k + 2) * U * each.abs().sum(1), "grad_x")

    y_rows = rows_of((n, width), dtype, seed + 2).requires_grad_(True)
    wdt = dict(f32=F32, same=dtype).get(weights)
    w = None if wdt is None else rows_of(experts.shape, wdt, seed + 3).requires_grad_(True)
    r = rows_of((*lead, width), dtype, seed + 4).requires_grad_(True) if residual else None
    y = combine_rows(y_rows, order, w, residual=r)
    assert y.shape == (*lead, width) and y.dtype == dtype
    e = y_rows.detach().double()[at] * there[:, None] if n else y_rows.detach().double()
    f = torch.ones(n, 1, dtype=torch.float64, device=DEV) if w is None else w.detach().double().reshape(-1, 1)
    terms = (e * f).view(-1, k, width)
    extra = r.detach().double().reshape(-1, width) if residual else 0.0
    close(y, terms.sum(1) + extra, (k + 3) * U * (terms.abs().sum(1) + (abs(extra) if residual else 0.0)), "y")
    dy = rows_of((*lead, width), dtype, seed + 5)
    names = [a for a, t in (("rows", y_rows), ("weights", w), ("residual", r)) if t is not None]
    grads = dict(zip(names, torch.autograd.grad(y, [t for t in (y_rows, w, r) if t is not None], dy)))
    spread = (dy.double().reshape(-1, 1, width) * f.view(-1, k, 1)).reshape(n, width)
    value = torch.zeros(n, width, dtype=torch.float64, device=DEV)
    value[flat[there]] = spread[there]
    close(grads["rows"], value, U * value.abs(), "grad_rows")
    if w is not None:
        prod = e.view(-1, k, width) * dy.double().reshape(-1, 1, width)
        close(grads["weights"], prod.sum(-1), (width + 2) * U * prod.abs().sum(-1), "grad_weights")
        assert grads["weights"].dtype == wdt
    if residual:
        assert torch.equal(grads["residual"], dy)


def experts_of(tokens, k, n_experts, none=0.1, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    e = torch.randint(0, n_experts, (tokens, k), generator=gen, device=DEV)
    return torch.where(torch.rand(tokens, k, generator=gen, device=DEV) < none, -1, e)


@pytest.mark.parametrize("tokens,k,n_experts", [(1, 1, 1), (1, 2, 24), (4, 2, 24), (7, 32, 3), (31, 1, 5), (33, 3, 2), (200, 4, 16), (683, 3, 7), (1023, 2, 64),
                                                (1024, 2, 64), (1025, 2, 64), (2048, 1, 300), (2500, 5, 1024), (9000, 8, 100)])
def test_orders(tokens, k, n_experts):
    for i, none in enumerate((0.0, 0.3, 1.0)):
        check_rows(experts_of(tokens, k, n_experts, none, seed=i), n_experts, 24, BF16)


@pytest.mark.parametrize("width", [1, 2, 3, 4, 7, 8, 9, 16, 31, 33, 64, 99, 128, 131, 250, 256, 259, 512, 1000, 1030, 2048, 4097])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_row_widths(width, dtype):
    for i, (tokens, k) in enumerate(((1, 1), (13, 2), (45, 3), (6, 9))):
        check_rows(experts_of(tokens, k, 5, 0.2, seed=i), 5, width, dtype, weights=[None, "f32", "same"][(width + i) % 3], residual=(width + i) % 2 == 0)


def test_leading_dimensions_and_no_tokens():
    check_rows(experts_of(24, 3, 5).view(2, 3, 4, 3), 5, 40, F16)
    check_rows(experts_of(24, 3, 5)[0], 5, 40, F16)
    check_rows(experts_of(24, 3, 5)[:0], 5, 40, F16)


def test_all_entries_of_one_expert_and_of_none():
    for value, n_experts in ((0, 4), (3, 4), (1023, 1024), (-1, 4), (4, 4), (1 << 40, 4), (-(1 << 40), 4), (1 << 32, 4)):
        check_rows(torch.full((3000, 2), value, device=DEV), n_experts, 16, BF16)
    runs = (torch.arange(6000, device=DEV) // 1500).view(-1, 2)            # sorted already
    check_rows(runs, 4, 16, BF16)
    check_rows(3 - runs, 4, 16, BF16)                                       # the other way round


def test_the_same_expert_twice():
    experts = torch.tensor([[1, 1, 1], [0, 1, 0], [2, 2, -1]], device=DEV)
    check_rows(experts, 3, 20, F32)


def test_many_rows():
    check_rows(experts_of(70001, 4, 64, 0.02), 64, 64, BF16)
    check_rows(experts_of(30001, 2, 16, 0.02), 16, 259, F16)
    for n_experts in (7, 500):      # blocks that place their entries in several parts
        check_rows(experts_of(90001, 8, n_experts, 0.02), n_experts, 8, BF16, residual=False)


def test_row_strides():
    """Operands that are not contiguous or start off a 16-byte boundary."""
    experts = experts_of(60, 6, 5)[:, ::2]
    base = torch.zeros(60 * 40 + 1, dtype=BF16, device=DEV)
    for x in (rows_of((40, 60), BF16).t(), base[1:].view(60, 40).copy_(rows_of((60, 40), BF16)), rows_of((1, 40), BF16).expand(60, 40)):
        rows, order = dispatch_rows(x, experts, 5)
        again, other = dispatch_rows(x.contiguous().clone(), experts.contiguous(), 5)
        assert torch.equal(rows, again) and torch.equal(order.position, other.position)
    w = rows_of((3, 60), F32).t()
    y = combine_rows(rows_of((40, 180), BF16).t(), order, w, residual=x)
    assert torch.equal(y, combine_rows(rows_of((40, 180), BF16).t().contiguous(), order, w.contiguous(), residual=x.contiguous()))
    leaf = rows_of((180, 40), BF16).requires_grad_(True)
    dy = rows_of((1, 40), BF16)
    (g,) = torch.autograd.grad(combine_rows(leaf, order, w), leaf, dy.expand(60, 40))
    (h,) = torch.autograd.grad(combine_rows(leaf, order, w), leaf, dy.expand(60, 40).contiguous())
    assert torch.equal(g, h)


def test_rows_of_nan_stay_where_they_are():
    """A padded token's row and the rows behind the last expert's reach nothing."""
    experts = experts_of(50, 2, 4, 0.0)
    experts[7] = -1
    x = rows_of((50, 24), F32)
    x[7] = NAN
    rows, order = dispatch_rows(x, experts, 4)
    assert torch.isfinite(rows).all() and not rows[98:].any()
    poisoned = rows.clone()
    poisoned[98:] = NAN
    poisoned.requires_grad_(True)
    w = torch.rand(50, 2, device=DEV, requires_grad=True)
    y = combine_rows(poisoned, order, w)
    assert torch.isfinite(y).all() and not y[7].any()
    gr, gw = torch.autograd.grad(y, (poisoned, w), torch.ones_like(y))
    assert torch.isfinite(gr).all() and torch.isfinite(gw).all() and not gr[98:].any() and not gw[7].any()


def test_row_gradients_against_differences():
    """Of dispatch and combine together, along a direction of everything that has a gradient; the sums are of products of two, so central
    differences in 64 bits have no error but rounding."""
    experts = experts_of(40, 3, 5, 0.2)
    leaves = [rows_of((40, 24), F32).requires_grad_(True), rows_of((40, 3), F32, 1).requires_grad_(True), rows_of((40, 24), F32, 2).requires_grad_(True)]
    factor, dy = rows_of((120, 24), F32, 3), rows_of((40, 24), F32, 4)
    rows, order = dispatch_rows(leaves[0], experts, 5)
    grads = torch.autograd.grad(combine_rows(rows * factor, order, leaves[1], residual=leaves[2]), leaves, dy)
    position = order_of(experts, 5)[1]
    there, at = (position >= 0)[..., None], position.clamp_min(0)

    def value(x, w, r):
        return (((x[:, None] * factor.double()[at]) * there * w[..., None]).sum(1) + r).mul(dy.double()).sum()

    moves = [torch.randn(t.shape, dtype=torch.float64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(i)) for i, t in enumerate(leaves)]
    up, down = (value(*(t.detach().double() + h * v for t, v in zip(leaves, moves))).item() for h in (0.5, -0.5))
    got = sum((g.double() * v).sum().item() for g, v in zip(grads, moves))
    # each gradient is a sum of at most 24 products of three factors, rounded at each
    size = sum((g.double().abs() * v.abs()).sum().item() for g, v in zip(grads, moves))
    terms = ((leaves[0].abs().double()[:, None] * factor.abs().double()[at]) * there * dy.abs().double()[:, None]).sum(-1)
    slack = 32 * U * (size + (terms * moves[1].abs()).sum().item())
    slack += 32 * U * ((factor.abs().double()[at] * there * leaves[1].detach().abs().double()[..., None]).sum(1) * dy.abs().double() * moves[0].abs()).sum().item()
    assert abs(got - (up - down)) <= slack + 1e-12 * size


def test_positions_that_lead_nowhere():
    """An order put together by hand with indices outside the rows: they count as none."""
    rows = rows_of((12, 16), F32).requires_grad_(True)
    position = torch.tensor([[0, 12], [-5, 3], [1 << 40, 4], [-(1 << 40), 11], [2, 1], [9, 10]], device=DEV)
    starts = torch.tensor([0, 1 << 50], device=DEV)
    w = torch.rand(6, 2, device=DEV, requires_grad=True)
    y = combine_rows(rows, (starts, position), w)
    at = torch.where((position >= 0) & (position < 12), position, -1)
    e = rows.detach().double()[at.clamp_min(0)] * (at >= 0)[..., None] * w.detach().double()[..., None]
    close(y, e.sum(1), 4 * U * e.abs().sum(1))
    gr, gw = torch.autograd.grad(y, (rows, w), torch.ones_like(y))
    assert torch.equal(gw == 0, at < 0)
    expected = torch.zeros(12, device=DEV).index_add_(0, at[at >= 0], w.detach()[at >= 0])  # no row twice: nothing is rounded
    assert torch.equal(gr, expected[:, None].expand(12, 16))


@pytest.mark.parametrize("tokens,k,width,dtype", [(1, 1, 8, F32), (40, 3, 24, BF16), (700, 2, 99, F32), (60, 4, 1031, F16), (60, 4, 4096, BF16),
                                                  (30000, 4, 64, BF16), (30000, 4, 35, BF16)])
def test_entries_taken_out_of_an_order(tokens, k, width, dtype):
    """Beyond an expert's capacity: the rows that no entry leads to any more get a gradient of 0 wherever they lie, the others theirs."""
    experts = experts_of(tokens, k, 7, 0.1)
    rows, order = dispatch_rows(rows_of((tokens, width), dtype), experts, 7)
    capacity = max(1, tokens * k // 11)
    beyond = order.position - order.group_start_index[experts.clamp(0, 6)] >= capacity
    kept = order._replace(position=order.position.masked_fill(beyond, -1))
    leaf, w, dy = rows.detach().requires_grad_(True), rows_of((tokens, k), F32, 1).requires_grad_(True), rows_of((tokens, width), dtype, 2)
    junk = [torch.full_like(rows, NAN) for _ in range(2)]  # what the gradient's memory may hold
    del junk
    gr, gw = torch.autograd.grad(combine_rows(leaf, kept, w), (leaf, w), dy)
    all_r, all_w = torch.autograd.grad(combine_rows(leaf, order, w), (leaf, w), dy)
    there = torch.zeros(tokens * k, dtype=torch.bool, device=DEV)
    there[kept.position[kept.position >= 0]] = True
    assert torch.equal(gr, torch.where(there[:, None], all_r, torch.zeros_like(all_r)))
    assert torch.equal(gw, all_w.masked_fill(kept.position < 0, 0.0))


def test_residual_of_another_type_keeps_its_bits():
    experts = experts_of(30, 2, 4, 0.0)
    rows, order = dispatch_rows(rows_of((30, 16), BF16), experts, 4)
    r = rows_of((30, 16), F32).requires_grad_(True)
    y = combine_rows(rows, order, residual=r)
    assert y.dtype == F32 and torch.equal(y, combine_rows(rows, order).float() + r)
    (g,) = torch.autograd.grad(y, r, torch.ones_like(y))
    assert torch.equal(g, torch.ones_like(r))


def test_functions_are_the_nodes():
    class Route(RouteExpertsFunction):
        pass

    class Dispatch(DispatchRowsFunction):
        pass

    class Combine(CombineRowsFunction):
        pass

    logits, x, dy = logits_of(90, 24), rows_of((90, 40), BF16), rows_of((90, 40), BF16, 1)
    out = []
    for route, dispatch, combine in ((RouteExpertsFunction, DispatchRowsFunction, CombineRowsFunction), (Route, Dispatch, Combine)):
        leaves = [t.detach().requires_grad_(True) for t in (logits, x)]
        w, e = route.apply(leaves[0], None, 3, 0, 1, 1, 0, False, 1.0)
        rows, starts, position = dispatch.apply(leaves[1], e, 24)
        y = combine.apply(rows, position, w, leaves[1])
        assert not e.requires_grad and not starts.requires_grad and not position.requires_grad
        out.append([w, e, rows, starts, position, y, *torch.autograd.grad(y, leaves, dy)])
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_no_second_derivative():
    leaf = logits_of(9, 24).requires_grad_(True)
    (g,) = torch.autograd.grad(route_experts(leaf, 3)[0].sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        g.sum().backward()


# ---- together -----------------------------------------------------------------------------------------------------------------
def dense_block(m, x, mask, logits_dtype=torch.float64):
    """``ExpertFeedForward`` by its definition in 64 bits, every expert for every token."""
    p = {n: t.double() for n, t in m.named_parameters()}
    h = torch.nn.functional.layer_norm(x, (x.shape[-1],), p["norm.weight"], p["norm.bias"], m.norm.eps)
    logits = h @ p["router"].t()
    experts = chosen(logits, m.top_k, m.balance, **m.routing)
    s = torch.softmax(logits, -1) if m.routing["score"] == "softmax" else torch.sigmoid(logits)
    c = s.gather(-1, experts)
    w = m.routing["scale"] * (c / c.sum(-1, keepdim=True) if m.routing["renormalise"] else c)
    every = torch.nn.functional.gelu(torch.einsum("...k,enk->...en", h, p["experts.weight1"]) + p["experts.bias1"])
    every = torch.einsum("...en,ekn->...ek", every, p["experts.weight2"]) + p["experts.bias2"]
    mine = every.gather(-2, experts[..., None].expand(*experts.shape, x.shape[-1]))
    return x + (w[..., None] * mine).sum(-2) * ~mask[..., None], experts


@pytest.mark.parametrize("options", [dict(), dict(score="sigmoid", balanced=True, n_groups=4, top_groups=2, group_score="top2", scale=2.5),
                                     dict(renormalise=False)], ids=str)
def test_block_of_experts(options):
    """Norm, router, experts and sum as one layer, forward and backward, fp32.  The products' sums have at most 128 terms and pass
    on errors of the norm's 32: each stage is off by less than 2^-16 of its magnitude (256 u), and there are six; gradients pass twice as many."""
    torch.manual_seed(1)
    m = ExpertFeedForward(32, 64, 8, 2, **options).to(DEV)
    for q in m.parameters():
        torch.nn.init.normal_(q, std=0.4)
    if m.balance is not None:
        m.balance.copy_(torch.randn(8) * 0.05)
    x = torch.randn(3, 50, 32, device=DEV, requires_grad=True)
    mask = torch.rand(3, 50, device=DEV) < 0.2
    y, order = m(x, mask, return_order=True)
    x64 = x.detach().double().requires_grad_(True)
    want, experts = dense_block(m, x64, mask)
    counts = torch.stack([((experts == e) & ~mask[..., None]).sum() for e in range(8)])
    assert torch.equal(order.group_start_index.diff(), counts)
    assert (y - want).abs().max() <= 6 * 2.0 ** -16 * want.abs().max()
    dy = torch.randn_like(y)
    leaves, names = [x, *m.parameters()], ["x", *dict(m.named_parameters())]
    got = torch.autograd.grad(y, leaves, dy)
    ref = torch.autograd.grad(want, [x64, *m.parameters()], dy.double())
    for name, a, b in zip(names, got, ref):
        assert (a - b).abs().max() <= 12 * 2.0 ** -16 * b.abs().max(), name


def test_block_without_tokens():
    m = ExpertFeedForward(32, 64, 8, 2).to(DEV)
    x = torch.zeros(2, 0, 32, device=DEV, requires_grad=True)
    y, order = m(x, return_order=True)
    assert y.shape == x.shape and not order.group_start_index.any()
    y.sum().backward()
    assert all(not p.grad.any() for p in m.parameters())
    y, order = m(torch.randn(5, 32, device=DEV), torch.ones(5, dtype=torch.bool, device=DEV), return_order=True)    # padding only
    assert not order.group_start_index.any() and (order.position == -1).all()


@pytest.mark.parametrize("tokens", [1, 3, 300])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_block_in_16_bits_follows_its_parts(dtype, tokens):
    """The module is its parts: the same bits as the calls one by one, fp32 parameters beside 16-bit rows."""
    from ops3d_b200 import fused_linear, layer_norm

    torch.manual_seed(2)
    m = ExpertFeedForward(64, 128, 8, 2).to(DEV)
    x = torch.randn(tokens, 64, device=DEV).to(dtype)
    with torch.no_grad():
        y, order = m(x, return_order=True)
        h = layer_norm(x, m.norm.weight, m.norm.bias)
        w, e = route_experts(fused_linear(h, m.router.to(dtype)), 2)
        rows, again = dispatch_rows(h, e, 8)
        hidden = grouped_linear(rows, m.experts.weight1.to(dtype), again.group_start_index, m.experts.bias1.to(dtype), activation="gelu")
        out = grouped_linear(hidden, m.experts.weight2.to(dtype), again.group_start_index, m.experts.bias2.to(dtype))
        assert torch.equal(y, combine_rows(out, again, w, residual=x)) and torch.equal(order.position, again.position)
    with torch.autocast("cuda", dtype=dtype):
        z = m(x.float())
        assert z.dtype == F32 and torch.isfinite(z).all()
        z.sum().backward()
    assert all(q.grad is not None and q.grad.dtype == F32 for q in m.parameters())


def test_captured_block_follows_its_inputs():
    """Choices, groups and rows change between replays of one graph."""
    torch.manual_seed(3)
    m = ExpertFeedForward(64, 128, 8, 2).to(DEV)
    x = torch.randn(97, 64, device=DEV, requires_grad=True)
    dy = torch.randn(97, 64, device=DEV)
    leaves = [x, *m.parameters()]

    def run():
        y = m(x)
        return [y, *torch.autograd.grad(y, leaves, dy)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            run()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = run()
    for seed in (4, 5):
        torch.manual_seed(seed)
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
            dy.copy_(torch.randn_like(dy))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, run()))


def test_repeated_calls_streams_and_threads():
    cases = [(logits_of(5000 + i, 64, BF16, seed=i), rows_of((5000 + i, 99), BF16, i), rows_of((5000 + i, 99), BF16, 9 + i)) for i in range(4)]

    def run(case):
        logits, x = (t.detach().requires_grad_(True) for t in case[:2])
        w, e = route_experts(logits, 4, bias=torch.zeros(64, device=DEV), score="sigmoid")
        rows, order = dispatch_rows(x, e, 64)
        y = combine_rows(rows, order, w, residual=x)
        return [w, e, rows, *order, y, *torch.autograd.grad(y, (logits, x), case[2])]

    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i] = run(cases[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_more_than_2_31_elements():
    """Offsets beyond 32 bits in rows, logits and gradients."""
    tokens, width = (1 << 23) + 3, 260
    experts = torch.zeros(tokens, 1, dtype=torch.int64, device=DEV)
    experts[-40:, 0] = 1
    x = torch.zeros(tokens, width, dtype=BF16, device=DEV)
    x[-40:] = rows_of((40, width), BF16)
    rows, order = dispatch_rows(x, experts, 2)
    assert order.group_start_index.tolist() == [0, tokens - 40, tokens] and torch.equal(rows, x)
    rows.requires_grad_(True)
    y = combine_rows(rows, order)
    assert torch.equal(y, x)
    (g,) = torch.autograd.grad(y, rows, x)
    assert torch.equal(g, x)
    logits = torch.zeros(tokens, 260, dtype=BF16, device=DEV)
    logits[-40:] = logits_of(40, 260, BF16)
    logits.requires_grad_(True)
    w, e = route_experts(logits, 2)
    assert torch.equal(e[-40:], chosen(logits[-40:].detach(), 2)) and not e[:100, 0].any()
    (g,) = torch.autograd.grad(w, logits, torch.ones_like(w) * torch.tensor([1.0, -1.0], device=DEV))
    value, bound = weights_of(logits[-40:].detach(), e[-40:], dw=torch.tensor([[1.0, -1.0]], device=DEV).expand(40, 2))["grad"]
    close(g[-40:], value, bound)
