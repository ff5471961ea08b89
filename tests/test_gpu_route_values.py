"""Routing of tokens whose logits are not ordinary numbers: NaN beside minus infinity, and sigmoid scores below fp32's range.

What NaN and minus infinity are worth is the operator's definition: a NaN compares as minus infinity, ties go to the lower index, and a
NaN that is chosen is one in the weights.
"""
import itertools

import pytest
import torch

from ops3d_b200 import route_experts

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF, NAN = float("inf"), float("nan")
U = 2.0 ** -24


def plain_choice(logits, k, bias, score, n_groups, top_groups, group_score):
    """One token's experts by the definition, in 64 bits on the host."""
    l = logits.double()
    s = torch.softmax(l, 0) if score == "softmax" else torch.sigmoid(l)
    if (l == -INF).all():
        s = torch.zeros_like(l)

    def worth_of(v):
        return [-INF if x != x else x + 0.0 for x in v.tolist()]

    sums = group_score == "top2" and len(l) > n_groups and top_groups < n_groups
    by_group = worth_of(s if bias is None and sums else l if bias is None else s + bias.double())
    by_expert = worth_of(l if bias is None else s + bias.double())
    size = len(l) // n_groups
    groups = range(n_groups)
    if top_groups < n_groups:
        def group(g):
            each = sorted(by_group[g * size:(g + 1) * size], reverse=True)
            return each[0] + each[1] if sums else each[0]
        groups = sorted(groups, key=lambda g: (-group(g), g))[:top_groups]
    left = [e for g in groups for e in range(g * size, (g + 1) * size)]
    return sorted(left, key=lambda e: (-by_expert[e], e))[:k]


def odd_logits(tokens, experts, seed):
    """Some tokens of finite logits, some of minus infinity and NaN but for a few."""
    gen = torch.Generator().manual_seed(seed)
    logits = torch.randn(tokens, experts, generator=gen) * 1.5
    kind = torch.rand(tokens, experts, generator=gen)
    share = torch.rand(tokens, 1, generator=gen)
    logits = torch.where(kind < share * 0.5, torch.tensor(NAN), torch.where(kind < share, torch.tensor(-INF), logits))
    logits[0], logits[1], logits[2] = NAN, -INF, torch.where(torch.arange(experts) % 2 == 0, NAN, -INF)
    logits[3, :-1] = torch.where(torch.arange(experts - 1) % 3 == 0, NAN, -INF)
    return logits


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("experts,k", [(3, 2), (24, 8), (40, 16), (64, 6), (100, 32), (256, 8), (300, 32), (600, 32)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_nan_beside_minus_infinity(score, experts, k, dtype):
    logits = odd_logits(43, experts, experts).to(dtype)
    off = torch.where(torch.arange(experts) % 5 == 1, -INF, 0.125 * (torch.arange(experts) % 3))
    for bias in (None, torch.zeros(experts), off):
        for n_groups, top_groups, group_score in ((1, 1, "max"), (2, 1, "max"), (4, 3, "top2")):
            if experts % n_groups or k > experts // n_groups * top_groups:
                continue
            args = (score, n_groups, top_groups, group_score)
            weights, chosen = route_experts(logits.to(DEV), k, bias=None if bias is None else bias.to(DEV), score=score, n_groups=n_groups,
                                            top_groups=top_groups, group_score=group_score, renormalise=False)
            want = torch.tensor([plain_choice(row, k, bias, *args) for row in logits])
            assert torch.equal(chosen.cpu(), want), (bias is not None, n_groups, (chosen.cpu() != want).any(-1).nonzero()[:, 0].tolist())
            assert weights.cpu()[logits.gather(1, want).isnan()].isnan().all()


def test_a_nan_takes_its_place_among_minus_infinities():
    logits = torch.tensor([[NAN, -INF, 5.0, -INF], [-INF, NAN, -INF, 5.0], [-INF, -INF, NAN, -INF]], device=DEV)
    for score in ("softmax", "sigmoid"):
        weights, chosen = route_experts(logits, 2, score=score)
        assert chosen.tolist() == [[2, 0], [3, 0], [0, 1]]
        assert weights[0].isnan().all()                   # the sum has the NaN in it
        assert weights[1].tolist() == [1.0, 0.0] and weights[2].tolist() == [0.0, 0.0]


# ---- sigmoid scores below fp32's range -----------------------------------------------------------------------------------------
def sigmoid_weights(logits, scale):
    """Renormalised sigmoid weights of the logits, in 64 bits by their logarithms: e^(log s_j) / sum, log s = -log(1 + e^-l)."""
    log_s = -torch.nn.functional.softplus(-logits, threshold=40.0)
    return scale * torch.softmax(log_s, -1)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("middle", [0.0, -20.0, -80.0, -87.0, -90.0, -100.0, -104.0, -300.0, -3e4])
@pytest.mark.parametrize("biased", [False, True])
def test_sigmoid_weights_of_any_logits(middle, biased, dtype):
    """Weights are ratios of scores, so they do not vanish with them.  With m = min(0, largest chosen logit) and far the largest l - m of a
    token's chosen, a score e^(l - m) / (1 + e^(l - m) e^m) is off by u (far + 4) above, u (far + 9) below the line, 2 u for sum and
    quotient; a weight by twice that and 12 u.  Gradients: their terms' magnitudes times three times that and 20 u."""
    gen = torch.Generator(device=DEV).manual_seed(int(-middle))
    logits = (middle + torch.randn(50, 40, generator=gen, device=DEV) * 2).to(dtype)
    logits[7, 1:] = -INF                                # a single one is left, and beside it scores of 0
    if dtype == F32:
        logits[8] = middle + torch.linspace(0, 3, 40, device=DEV)
    bias = torch.linspace(1.0, 0.0, 40, device=DEV) if biased else None
    for k, scale in ((1, 1.0), (4, 2.5), (20, 1.0)):
        leaf = logits.detach().requires_grad_(True)
        weights, experts = route_experts(leaf, k, bias=bias, score="sigmoid", scale=scale)
        l = logits.double().gather(1, experts)
        l64 = l.clone().requires_grad_(True)
        want = sigmoid_weights(l64, scale)
        top = l.max(-1, keepdim=True).values.clamp(max=0)
        far = torch.where((l < 0) & (l > -INF), (l - top).abs(), torch.zeros_like(l)).max(-1, keepdim=True).values
        rel = (2 * (2 * far + 15) + 12) * U
        bound = want.detach() * rel + 2.0 ** -125
        assert ((weights.double() - want.detach()).abs() <= bound).all()
        assert (weights.double().sum(-1) - scale).abs().max() <= scale * 40 * U
        dw = torch.randn(50, k, generator=gen, device=DEV)
        (grad,) = torch.autograd.grad(weights, leaf, dw)
        share, d = want.detach() / scale, dw.double() * scale
        slope = torch.sigmoid(-l)
        value = share * (d - (d * share).sum(-1, keepdim=True)) * slope
        # the formula is the reference's own derivative, minus infinities (whose logarithm has none) aside
        (auto,) = torch.autograd.grad(want, l64, dw.double())
        there = (l > -INF).all(-1)
        assert (auto - value)[there].abs().max() <= 1e-12 * d.abs().max()
        magnitude = share * (d.abs() + (d.abs() * share).sum(-1, keepdim=True)) * slope
        fi = torch.finfo(dtype)
        allowed = magnitude * (3 * rel + 20 * U) + value.abs() * (fi.eps / 2) * 1.02 + fi.tiny * fi.eps / 2 + 2.0 ** -125
        got = grad.double().gather(1, experts)
        assert ((got - value).abs() <= allowed).all()
        assert not grad.scatter(1, experts, 0.0).any()


def test_sigmoid_gradient_against_differences_at_low_logits():
    """At -95 the quotient of differences of the 64-bit weights and the gradient agree.  For values of order 1 the quotient's own error is
    h^2 times a third derivative below 1: 2^-16 is far above it and far below the gradients."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    logits = (-95 + torch.randn(9, 12, generator=gen, device=DEV)).requires_grad_(True)
    weights, experts = route_experts(logits, 3, score="sigmoid")
    dw = torch.randn(9, 3, generator=gen, device=DEV)
    (grad,) = torch.autograd.grad(weights, logits, dw)
    v = torch.randn(9, 12, generator=gen, device=DEV, dtype=torch.float64)
    h = 2.0 ** -10
    a, b = ((sigmoid_weights((logits.detach().double() + t * v).gather(1, experts), 1.0) * dw).sum() for t in (h, -h))
    assert abs((grad.double() * v).sum() - (a - b) / (2 * h)) <= 2.0 ** -16 * (v.abs().sum() + 1)
    assert (grad.abs().amax(-1) > 0).all()


@pytest.mark.parametrize("biased", [False, True])
def test_sigmoid_scores_down_to_the_smallest(biased):
    """Without renormalising a weight is the score: relative to it 8 u, and two steps of the smallest numbers."""
    logits = torch.linspace(-103, 90, 4 * 193, device=DEV).view(-1, 4)
    bias = torch.zeros(4, device=DEV) if biased else None
    weights, experts = route_experts(logits, 4, bias=bias, score="sigmoid", renormalise=False)
    want = torch.sigmoid(logits.double().gather(1, experts))
    assert ((weights.double() - want).abs() <= 8 * U * want + 2.0 ** -147).all()


def test_lowest_values_as_masks_share_the_weight():
    """Equal logits have equal weights whatever they are; only minus infinity is no score at all."""
    for dtype in (F32, F16, BF16):
        for value in (torch.finfo(dtype).min, -200.0):
            logits = torch.full((3, 24), value, dtype=dtype, device=DEV, requires_grad=True)
            weights, experts = route_experts(logits, 4, score="sigmoid")
            assert torch.equal(weights, torch.full_like(weights, 0.25)) and torch.equal(experts, torch.arange(4, device=DEV).expand(3, 4))
            (grad,) = torch.autograd.grad(weights, logits, torch.tensor([[1.0, 0, 0, 0]], device=DEV).expand(3, 4))
            assert torch.equal(grad[:, :4], torch.tensor([[0.1875, -0.0625, -0.0625, -0.0625]], dtype=dtype, device=DEV).expand(3, 4))
    mixed = torch.tensor([[-INF, torch.finfo(F32).min, -INF, -INF]], device=DEV)
    weights, experts = route_experts(mixed, 2, score="sigmoid")
    assert experts.tolist() == [[1, 0]] and weights.tolist() == [[1.0, 0.0]]
