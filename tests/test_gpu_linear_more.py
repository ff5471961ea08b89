"""Linear operators at the ends of their types' range, bias gradients at every width, waits' count, and autograd's other tools."""
import pytest
import torch

from ops3d_b200 import capi, fused_linear, grouped_linear
from test_gpu_linear import ACTS, DEV, DTYPES, act64, make, rounding

pytestmark = pytest.mark.gpu

NARROW = [torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    torch.cuda.synchronize()
    assert capi.load().fda_linear_timeouts() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_values_and_slopes_up_to_the_types_limit(act, dtype):
    """Far out the activations are v or 0 and their slopes 1 or 0 exactly, also where v^2 or v^3 overflows: beyond 128 the exponentials
    are 0 or above every fp32 number, and all that is left is one rounding."""
    top = torch.finfo(dtype).max
    v = torch.tensor([s * a for a in (128.0, 3e3, 6e4, 1e7, 1e13, 3e18, 1e20, 1e30, 2e38, top) if a <= top for s in (1, -1)], device=DEV)
    for copies in (1, 20, 2000):
        x = torch.zeros(v.numel() * copies, 8, device=DEV, dtype=dtype)
        x[:, 3] = v.repeat(copies).to(dtype)
        w = torch.zeros(16, 8, device=DEV, dtype=dtype)
        w[:, 3] = 1
        x.requires_grad_(True)
        y = fused_linear(x, w, activation=act)
        (gx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        at = x.detach()[:, 3]
        want = at if act == "none" else at.clamp_min(0)
        slope = torch.ones_like(at) if act == "none" else (at > 0).to(dtype)
        assert torch.equal(y, want[:, None].expand_as(y))
        assert torch.equal(gx[:, 3], 16 * slope) and not gx[:, :3].any() and not gx[:, 4:].any()


@pytest.mark.parametrize("dtype", NARROW)
@pytest.mark.parametrize("groups,M,K,N", [(1, 300, 40, 1024), (1, 3000, 33, 1027), (1, 19003, 72, 1024), (1, 5003, 40, 2056), (16, 9000, 72, 264),
                                          (70, 4000, 24, 136), (2, 30000, 40, 520)])
def test_bias_gradient_is_rounded_once_at_every_width(groups, M, K, N, dtype):
    """The precision of a bias's gradient does not depend on how many biases there are: fp32 sums of unrounded terms, one rounding.  (fp32's
    share as in test_bias_gradient_is_rounded_once: sums over 32 rows, of which a warp adds every 32nd.)"""
    x, w, b, _, dy = make((M,), K, N, dtype, groups, residual=False, seed=M)
    cuts = torch.sort(torch.randint(0, M, (groups - 1,), generator=torch.Generator().manual_seed(groups)))[0].tolist()
    bounds = [0, *cuts, M]
    leaf = b.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(grouped_linear(x, w, torch.tensor(bounds, device=DEV), leaf, activation="silu"), leaf, dy)
    for e in range(groups):
        rows = slice(bounds[e], bounds[e + 1])
        terms = dy[rows].double() * act64(x[rows].double() @ w[e].double().t() + b[e].double(), "silu")[1]
        value = terms.sum(0)
        slack = terms.abs().sum(0) * 2.0 ** -23 * 96 + dy[rows].double().abs().sum(0) * 2.0 ** -20 * 4
        assert ((g[e].double() - value).abs() <= rounding(value, dtype) * 1.01 + slack).all(), e


def test_counting_waits_waits_for_every_stream():
    """The count is asked for when nothing runs any more, on streams too that do not wait for the default one."""
    side = torch.cuda.Stream()
    x, w = (torch.ones(n, 64, device=DEV, dtype=torch.bfloat16) for n in (300, 64))
    fused_linear(x, w)              # what a first call loads is loaded
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)
        y = fused_linear(x, w)
    assert not side.query()
    assert capi.load().fda_linear_timeouts() == 0
    assert side.query()
    assert torch.equal(y, torch.full_like(y, 64))


def test_saved_tensor_hooks_see_what_the_backward_needs():
    """Tensors that hooks pack away and bring back, to the host for instance, give the same gradients."""
    x, w, b, r, dy = make((2, 150), 40, 56, torch.bfloat16, 3, seed=4)
    starts = torch.tensor([0, 20, 90], device=DEV)

    def grads():
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
        y = grouped_linear(leaves[0], leaves[1], starts, leaves[2], leaves[3], "gelu")
        return torch.autograd.grad(y, leaves, dy)

    want = grads()
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t.shape) or t.cpu(), lambda t: t.to(DEV)):
        got = grads()
    assert sorted(map(len, packed)) == [1, 2, 3, 3]
    with torch.autograd.graph.save_on_cpu():
        again = grads()
    for a, c, e in zip(got, again, want):
        assert torch.equal(a, e) and torch.equal(c, e)


def test_function_transforms_are_refused():
    """torch.func has no rule for the operators; it says so, and nothing is computed from a wrapper's storage."""
    x, w, b, _, _ = make((10,), 16, 24, torch.float32)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: fused_linear(t, w, b).sum())(x)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: fused_linear(t, w, b))(x[None].expand(3, 10, 16))
    with pytest.raises(RuntimeError):
        torch.func.jacrev(lambda t: fused_linear(t, w, b))(x)
    y = fused_linear(x, w, b)                     # and the process is as it was
    assert torch.isfinite(y).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_layers_saved_before_the_level_projections(dtype):
    """A whole layer pickled by an earlier version has no attribute for them."""
    from ops3d_b200.msda3d import MSDeformAttn3D

    layer = MSDeformAttn3D(32, 1, 4, 4).to(DEV, dtype)
    shapes, lsi = torch.tensor([(3, 4, 5)], device=DEV), torch.tensor([0], device=DEV)
    src, ref = torch.randn(2, 60, 32, device=DEV).to(dtype), torch.rand(2, 60, 1, 3, device=DEV)
    want = layer(src, ref, src, shapes, lsi)
    del layer.__dict__["level_value_proj"]
    assert torch.equal(layer(src, ref, src, shapes, lsi), want)


def test_no_wait_runs_out():
    """The Python name of the count."""
    import ops3d_b200

    y = fused_linear(torch.ones(5000, 64, device=DEV, dtype=torch.bfloat16), torch.ones(264, 64, device=DEV, dtype=torch.bfloat16))
    assert ops3d_b200.linear_timeouts() == 0 and torch.equal(y, torch.full_like(y, 64))


def test_fp32_bias_gradient_adds_in_short_chains():
    """A one every 128 rows and terms that a sum of one swallows between them.  fp32 sums over 16 rows, 16 of these, and one addition: off by
    at most 33 roundings, 2^-24 each, of the sum of the magnitudes.  (A chain of 128 loses 127 terms of 2^-25 for every one: 64 such units.)"""
    gen = torch.Generator(device=DEV).manual_seed(0)
    dy = torch.full((256, 70), 2.0 ** -25, device=DEV)
    dy[::128] = 1
    x, w = torch.randn(256, 8, generator=gen, device=DEV), torch.randn(70, 8, generator=gen, device=DEV)
    b = torch.zeros(70, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(fused_linear(x, w, b), b, dy)
    value = dy.double().sum(0)
    assert ((g.double() - value).abs() <= 33 * 2.0 ** -24 * value + 2.0 ** -24 * value).all()
