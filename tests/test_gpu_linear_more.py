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
def test_layers_saved_before_the_level_projections(dtype):
    """A whole layer pickled by an earlier version has no attribute for them."""
    from ops3d_b200.msda3d import MSDeformAttn3D

    layer = MSDeformAttn3D(32, 1, 4, 4).to(DEV, dtype)
    shapes, lsi = torch.tensor([(3, 4, 5)], device=DEV), torch.tensor([0], device=DEV)
    src, ref = torch.randn(2, 60, 32, device=DEV).to(dtype), torch.rand(2, 60, 1, 3, device=DEV)
    want = layer(src, ref, src, shapes, lsi)
    del layer.__dict__["level_value_proj"]
    assert torch.equal(layer(src, ref, src, shapes, lsi), want)
