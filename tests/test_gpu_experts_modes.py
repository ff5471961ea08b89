"""Layer norm, routing and the rows sorted by expert inside what torch wraps around operators: hooks on saved tensors, function transforms,
recomputation, autocast."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from ops3d_b200 import ExpertFeedForward, combine_rows, dispatch_rows, fused_linear, grouped_linear, layer_norm, linear_timeouts, route_experts

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    assert linear_timeouts() == 0


def normal(*size, dtype=F32, seed=0):
    return torch.randn(*size, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def chain(x, weight, bias, residual, router):
    """Norm with its sum, routing, rows and back; every operator has a gradient to give."""
    h, s = layer_norm(x, weight, bias, residual=residual, return_sum=True)
    weights, experts = route_experts(fused_linear(h, router), 3, score="sigmoid")
    rows, order = dispatch_rows(h, experts, router.shape[0])
    return combine_rows(rows, order, weights, residual=s)


def inputs(dtype):
    return [normal(150, 40, dtype=dtype), normal(40, dtype=dtype, seed=1), normal(40, dtype=dtype, seed=2), normal(150, 40, dtype=dtype, seed=3),
            normal(24, 40, dtype=dtype, seed=4)]


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_saved_tensor_hooks_see_what_the_backward_needs(dtype):
    dy = normal(150, 40, dtype=dtype, seed=9)

    def grads():
        leaves = [t.clone().requires_grad_(True) for t in inputs(dtype)]
        return torch.autograd.grad(chain(*leaves), leaves, dy)

    want = grads()
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(tuple(t.shape)) or t.cpu(), lambda t: t.to(DEV)):
        got = grads()
    # norm: x, weight, bias, residual; router: h, its weight; routing: logits, experts; rows: position; sums: rows, position, weights
    assert sorted(packed) == sorted([(150, 40), (40,), (40,), (150, 40), (150, 40), (24, 40), (150, 24), (150, 3), (150, 3), (450, 40), (150, 3), (150, 3)])
    with torch.autograd.graph.save_on_cpu():
        again = grads()
    for a, c, e in zip(got, again, want):
        assert torch.equal(a, e) and torch.equal(c, e)


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed(reentrant):
    dy = normal(150, 40, dtype=BF16, seed=9)
    out = []
    for recompute in (False, True):
        leaves = [t.clone().requires_grad_(True) for t in inputs(BF16)]
        y = checkpoint(chain, *leaves, use_reentrant=reentrant) if recompute else chain(*leaves)
        y.backward(dy)
        out.append([y, *[t.grad for t in leaves]])
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_a_changed_input_is_noticed():
    """What the backward reads is checked for changes since the forward."""
    for i in range(5):
        leaves = [t.clone().requires_grad_(True) for t in inputs(F32)]
        y = chain(*leaves)
        with torch.no_grad():
            leaves[i].mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    weights, experts = route_experts(normal(9, 24).requires_grad_(True), 2)
    experts[0] = -1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        weights.sum().backward()


def test_function_transforms_are_refused():
    """torch.func has no rule for the operators; it says so, and nothing is computed from a wrapper's storage."""
    x, w, b, r, _ = inputs(F32)
    logits = normal(150, 24, seed=5)
    weights, experts = route_experts(logits, 2)
    rows, order = dispatch_rows(x, experts, 24)
    calls = [(lambda t: layer_norm(t, w, b), x), (lambda t: layer_norm(x, t, b), w), (lambda t: layer_norm(x, w, b, residual=t, return_sum=True)[0], r),
             (lambda t: route_experts(t, 2)[0], logits), (lambda t: dispatch_rows(t, experts, 24)[0], x), (lambda t: combine_rows(t, order, weights), rows),
             (lambda t: combine_rows(rows, order, t), weights), (lambda t: combine_rows(rows, order, weights, residual=t), x)]
    for call, t in calls:
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda v: call(v).sum())(t)
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(t[None].expand(3, *t.shape))
        with pytest.raises(RuntimeError):
            torch.func.jacrev(call)(t)
        assert torch.isfinite(call(t)).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("options", [dict(), dict(score="sigmoid", balanced=True, n_groups=4, top_groups=2, group_score="top2", scale=2.5),
                                     dict(renormalise=False, residual=False), dict(norm=False)], ids=str)
def test_block_under_autocast_follows_its_parts(options, dtype):
    """An fp32 stream around 16-bit products: the block's output and gradients are those of its parts called one by one."""
    torch.manual_seed(3)
    m = ExpertFeedForward(72, 136, 8, 2, **options).to(DEV)
    for q in m.parameters():
        torch.nn.init.normal_(q, std=0.2)
    if m.balance is not None:
        m.balance.copy_(torch.randn(8) * 0.05)
    x, dy = normal(3, 101, 72).requires_grad_(True), normal(3, 101, 72, seed=1)
    mask = torch.rand(3, 101, device=DEV) < 0.2
    with torch.autocast("cuda", dtype):
        y, order = m(x, mask, return_order=True)
    f = m.experts
    h = x if m.norm is None else layer_norm(x, m.norm.weight, m.norm.bias)
    weights, experts = route_experts(fused_linear(h.to(dtype), m.router.to(dtype)), 2, m.balance, **m.routing)
    rows, again = dispatch_rows(h, experts.masked_fill(mask[..., None], -1), 8)
    hidden = grouped_linear(rows.to(dtype), f.weight1.to(dtype), again.group_start_index, f.bias1.to(dtype), activation="gelu")
    out = grouped_linear(hidden, f.weight2.to(dtype), again.group_start_index, f.bias2.to(dtype))
    want = combine_rows(out, again, weights)
    if m.residual:
        want = want + x
    assert torch.equal(order.position, again.position) and torch.equal(order.group_start_index, again.group_start_index)
    assert y.dtype == (F32 if m.residual else dtype) and torch.equal(y, want)
    leaves = [x, *m.parameters()]
    for g, v in zip(torch.autograd.grad(y, leaves, dy.to(y.dtype)), torch.autograd.grad(want, leaves, dy.to(y.dtype))):
        assert g.dtype == F32 and torch.equal(g, v)
