"""Linear operators and the modules made of them beside tensors of another type: a residual stream in fp32 around a 16-bit layer, and
``torch.autocast``, under which they take the types that torch's own linear layers take.

Where two sides make the same product of the same 16-bit tensors in two kernels, each rounds the same sum once: they differ by at most
``eps`` of the value (two half steps), and by fp32's share of the sum.  A gradient that has passed n such steps differs by n ``eps`` in
the norm; 8 ``eps`` is asked for, with at most five steps on the way."""
import pytest
import torch

from oracle.fda_oracle import level_start_index_of
from ops3d_b200 import FeedForward, GroupedLinear, fused_linear, grouped_linear
from ops3d_b200.msda3d import MSDeformAttn3D

pytestmark = pytest.mark.gpu

DEV = "cuda"
NARROW = [torch.float16, torch.bfloat16]


def layer_and_inputs(dtype=torch.float32, **options):
    torch.manual_seed(0)
    shapes = torch.tensor([(6, 8, 10), (3, 4, 5)])
    lsi = level_start_index_of(shapes).to(DEV)
    N, C = int(shapes.prod(1).sum()), 64
    layer = MSDeformAttn3D(C, 2, 4, 4, **options).to(DEV)
    with torch.no_grad():
        layer.sampling_offsets.weight.normal_(0, 0.05)
        layer.attention_weights.weight.normal_(0, 0.3)
        for p in (layer.value_proj.bias, layer.output_proj.bias):
            p.normal_(0, 0.1)
    src = torch.randn(2, N, C, device=DEV).to(dtype).requires_grad_(True)
    ref = torch.rand(2, N, 2, 3, device=DEV)
    return layer.to(dtype), src, (ref, src, shapes.to(DEV), lsi)


def near(got, want, eps, slack=1e-5):
    assert got.dtype == want.dtype and got.shape == want.shape
    d = (got.detach().double() - want.detach().double()).abs()
    return bool((d <= eps * 1.01 * want.detach().double().abs() + slack).all())


def norm_error(got, want):
    return ((got.double() - want.double()).norm() / want.double().norm().clamp_min(1e-30)).item()


@pytest.mark.parametrize("dtype", NARROW)
def test_fp32_residual_around_a_16_bit_layer(dtype):
    """``residual=`` gives what adding outside gives: the stream keeps its type and its bits."""
    layer, src, rest = layer_and_inputs(dtype)
    stream = torch.randn(src.shape, device=DEV, requires_grad=True)
    dy = torch.randn(src.shape, device=DEV)
    eps = torch.finfo(dtype).eps
    leaves = [stream, src, *layer.parameters()]
    want_proj = layer(src, *rest)
    want = want_proj + stream
    got = layer(src, *rest, residual=stream)
    assert got.dtype == torch.float32
    assert near(got - stream, want_proj.float(), eps)
    for g, v in zip(torch.autograd.grad(got, leaves, dy), torch.autograd.grad(want, leaves, dy)):
        assert g.dtype == v.dtype and norm_error(g, v) <= 8 * eps
    assert torch.equal(torch.autograd.grad(layer(src, *rest, residual=stream), stream, dy)[0], dy)


@pytest.mark.parametrize("dtype", NARROW)
@pytest.mark.parametrize("levels", [False, True], ids=["one-projection", "level-projections"])
def test_layer_under_autocast(levels, dtype):
    """From an fp32 stream: the projections run in autocast's type, the residual stays fp32, every gradient comes back in fp32."""
    layer, src, rest = layer_and_inputs()
    eps = torch.finfo(dtype).eps
    dy = torch.randn(src.shape, device=DEV)
    leaves = [src, layer.sampling_offsets.weight, layer.attention_weights.bias, layer.output_proj.weight, layer.output_proj.bias]
    with torch.autocast("cuda", dtype):
        want_proj = layer(src, *rest)
        want = want_proj + src
    assert want_proj.dtype == dtype
    wants = torch.autograd.grad(want, leaves, dy)
    if levels:   # the same weight for every level
        torch.manual_seed(1)
        other = MSDeformAttn3D(64, 2, 4, 4, level_value_proj=True).to(DEV)
        state = layer.state_dict()
        for k in ("weight", "bias"):
            state["value_proj." + k] = state["value_proj." + k].expand(2, *state["value_proj." + k].shape).contiguous()
        other.load_state_dict(state)
        layer = other
        leaves = [src, layer.sampling_offsets.weight, layer.attention_weights.bias, layer.output_proj.weight, layer.output_proj.bias]
    seen = []
    hook = layer.value_proj.register_forward_hook(lambda m, i, o: seen.append(o.dtype))
    with torch.autocast("cuda", dtype):
        got = layer(src, *rest, residual=src)
    hook.remove()
    assert seen == [dtype] and got.dtype == torch.float32
    assert norm_error(got - src, want_proj) <= 8 * eps
    for g, v in zip(torch.autograd.grad(got, leaves, dy), wants):
        assert g.dtype == torch.float32 and norm_error(g, v) <= 8 * eps


@pytest.mark.parametrize("dtype", NARROW)
@pytest.mark.parametrize("n_groups", [None, 3])
def test_feed_forward_under_autocast(n_groups, dtype):
    """Behind a norm, whose result autocast leaves in fp32: both products in 16 bits, the residual in fp32."""
    torch.manual_seed(2)
    ff = FeedForward(72, 136, "gelu", n_groups).to(DEV)
    starts = None if n_groups is None else torch.tensor([0, 100, 180], device=DEV)
    x = torch.randn(300, 72, device=DEV, requires_grad=True)
    dy = torch.randn(300, 72, device=DEV)
    leaves = [x, *ff.parameters()]
    with torch.autocast("cuda", dtype):
        got = ff(x, starts)
    w1, b1, w2, b2 = (p.to(dtype) for p in (ff.weight1, ff.bias1, ff.weight2, ff.bias2))
    if n_groups is None:
        want = fused_linear(fused_linear(x.to(dtype), w1, b1, activation="gelu"), w2, b2) + x
    else:
        want = grouped_linear(grouped_linear(x.to(dtype), w1, starts, b1, activation="gelu"), w2, starts, b2) + x
    assert got.dtype == torch.float32 and torch.equal(got, want)
    for g, v in zip(torch.autograd.grad(got, leaves, dy), torch.autograd.grad(want, leaves, dy)):
        assert g.dtype == torch.float32 and torch.equal(g, v)


def test_functions_under_autocast():
    torch.manual_seed(3)
    x, w, b, r = (torch.randn(*s, device=DEV) for s in ((90, 40), (56, 40), (56,), (90, 56)))
    low = [t.bfloat16() for t in (x, w, b, r)]
    starts = torch.tensor([0, 30], device=DEV)
    with torch.autocast("cuda", torch.bfloat16):
        assert torch.equal(fused_linear(x, w, b, activation="silu"), fused_linear(*low[:3], activation="silu"))
        assert torch.equal(fused_linear(low[0], w, low[2], low[3]), fused_linear(*low))
        assert torch.equal(fused_linear(x, w, b, r), fused_linear(*low[:3]) + r)
        assert torch.equal(grouped_linear(x, w.expand(2, 56, 40), starts, None, r), grouped_linear(low[0], low[1].expand(2, 56, 40), starts) + r)
        lin = GroupedLinear(2, 40, 56).to(DEV)
        assert torch.equal(lin(x, starts), grouped_linear(low[0], lin.weight.bfloat16(), starts, lin.bias.bfloat16()))
        with pytest.raises(RuntimeError, match="shape of the output"):
            fused_linear(x, w, b, r[:1])
        with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
            fused_linear(x.double(), w.double())
        with torch.autocast("cuda", enabled=False):
            assert fused_linear(x, w, b, r).dtype == torch.float32
    with torch.autocast("cuda", torch.float16):   # tensors of the other 16-bit type too, as torch's own layers
        assert torch.equal(fused_linear(low[0], w, low[2]), fused_linear(low[0].half(), w.half(), low[2].half()))


def test_captured_and_recomputed_under_autocast():
    """One graph of a training pass from an fp32 stream, whose inputs change between replays, and the same pass inside a checkpoint."""
    from torch.utils.checkpoint import checkpoint

    torch.manual_seed(4)
    ff = FeedForward(40, 72, "silu", 3).to(DEV)
    starts = torch.tensor([0, 50, 130], device=DEV)
    x, dy = torch.randn(2, 200, 40, device=DEV, requires_grad=True), torch.randn(2, 200, 40, device=DEV)
    leaves = [x, *ff.parameters()]

    def step(recompute=False):
        with torch.autocast("cuda", torch.bfloat16):
            y = checkpoint(ff, x, starts, use_reentrant=False) if recompute else ff(x, starts)
        return (y, *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for boundaries in ([0, 50, 130], [10, 10, 200], [0, 0, 0]):
        with torch.no_grad():
            starts.copy_(torch.tensor(boundaries))
            x.copy_(torch.randn(2, 200, 40))
        graph.replay()
        torch.cuda.synchronize()
        for a, e, r in zip(out, step(), step(recompute=True)):
            assert a.dtype == torch.float32 and torch.equal(a, e) and torch.equal(r, e)
