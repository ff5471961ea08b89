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
