"""``ExpertFeedForward`` with padding: what padded tokens hold reaches nothing but their own row of the residual."""
import pytest
import torch

from ops3d_b200 import ExpertFeedForward, linear_timeouts

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    assert linear_timeouts() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("options", [dict(), dict(score="sigmoid", balanced=True, n_groups=4, top_groups=2, group_score="top2"), dict(renormalise=False),
                                     dict(norm=False), dict(residual=False)], ids=str)
def test_padding_may_hold_anything(options, autocast, dtype):
    if autocast and dtype != F32:
        pytest.skip("an fp32 stream")
    torch.manual_seed(5)
    m = ExpertFeedForward(40, 72, 8, 2, **options).to(DEV)
    dy = torch.randn(3, 50, 40, device=DEV)
    base = torch.randn(3, 50, 40, device=DEV).to(dtype)
    mask = torch.rand(3, 50, device=DEV) < 0.3
    mask[1] = True                                         # a sequence of nothing else
    out = []
    for value in (0.0, 3.0, float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min):
        x = base.masked_fill(mask[..., None], value).requires_grad_(True)
        with torch.autocast("cuda", BF16, enabled=autocast):
            y, order = m(x, mask, return_order=True)
        assert (order.position[mask] == -1).all() and (order.position[~mask] >= 0).all()
        grads = torch.autograd.grad(y, [x, *m.parameters()], dy.to(y.dtype))
        if m.residual:
            assert torch.equal(grads[0][mask], dy.to(y.dtype)[mask].to(dtype))
            assert torch.equal(y[mask], x.detach()[mask].to(y.dtype)) or value != value
        else:
            assert not y[mask].any() and not grads[0][mask].any()
        out.append([y[~mask], grads[0][~mask], *grads[1:]])
        assert all(torch.isfinite(t).all() for t in out[-1])
        assert all(torch.equal(a, b) for a, b in zip(out[0], out[-1])), value
