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
