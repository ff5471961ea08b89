"""Host side of the linear operators: what the C ABI and the Python entry points refuse before a kernel is launched, how large the
workspaces are, and what has to see the autograd Function.  No device needed."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import ops3d_b200
import ops3d_b200.linear as linear_mod
from ops3d_b200 import capi

P = ctypes.c_void_p(256)


def _forward(lib, ptr=P, starts=None, num_starts=0, batch=1, rows=4, groups=1, k=8, n=8, act=0, dtype=2):
    return lib.fda_linear_forward(ptr, ptr, ptr, ptr, starts, num_starts, ptr, None, 0, batch, rows, groups, k, n, act, dtype, None)


def _backward(lib, ptr=P, starts=None, num_starts=0, ws=P, ws_bytes=1 << 40, batch=1, rows=4, groups=1, k=8, n=8, act=0, dtype=2):
    return lib.fda_linear_backward(ptr, ptr, ptr, ptr, starts, num_starts, ptr, ptr, ptr, ws, ws_bytes, batch, rows, groups, k, n, act,
                                   dtype, None)


@pytest.mark.parametrize("call", [_forward, _backward])
def test_arguments_are_checked_on_the_host(call):
    lib = capi.load()
    assert call(lib, dtype=3) == 2 and call(lib, dtype=-1) == 2
    assert call(lib, k=0) == 6 and call(lib, n=0) == 6 and call(lib, groups=0) == 6 and call(lib, rows=-1) == 6 and call(lib, batch=-1) == 6
    assert call(lib, batch=1 << 16, rows=1 << 15) == 6            # rows are counted in 31 bits
    assert call(lib, k=1 << 26) == 6 and call(lib, n=1 << 26) == 6
    assert call(lib, act=5) == 12 and call(lib, act=-1) == 12
    assert lib.fda_status_string(12) == b"unknown activation"
    assert call(lib, groups=1025, starts=P, num_starts=1025) == 11
    assert call(lib, groups=2) == 1                               # several groups without their start indices
    assert call(lib, groups=2, starts=P, num_starts=1) == 6 and call(lib, groups=2, starts=P, num_starts=4) == 6
    assert call(lib, ptr=None) == 1


def test_no_rows_no_launch():
    lib = capi.load()
    assert _forward(lib, rows=0) == 0 and _forward(lib, batch=0) == 0


def test_workspaces_hold_what_the_sizes_need():
    """Odd widths need padded copies, an activation the pre-activation's gradient, few rows only that in fp32, none at all where
    nothing is kept."""
    lib = capi.load()
    fwd, bwd = lib.fda_linear_forward_workspace_bytes, lib.fda_linear_backward_workspace_bytes
    assert fwd(1, 1000, 1, 64, 64, 2) == 0 and fwd(1, 1000, 1, 63, 64, 0) == 0 and fwd(1, 8, 1, 63, 64, 2) == 0
    assert fwd(1, 1000, 1, 63, 64, 2) >= 1000 * 64 * 2 + 64 * 64 * 2
    assert bwd(1, 64, 1, 63, 50, 0, 2) == 0 and 64 * 50 * 4 <= bwd(1, 64, 1, 63, 50, 2, 2) < 64 * 50 * 4 + 256
    assert bwd(1, 65, 1, 64, 64, 0, 2) == 0                       # one piece: no partial sums
    assert bwd(1, 65, 1, 64, 50, 0, 2) >= 65 * 56 * 2             # a padded copy of grad_output
    big = bwd(2, 300000, 3, 256, 256, 0, 2)
    assert big % (256 * 256 * 4 + 256 * 4) < 512 and big > 30 * 256 * 256 * 4   # slots of partial sums


def test_backward_workspace_is_checked():
    lib = capi.load()
    need = lib.fda_linear_backward_workspace_bytes(1, 100, 1, 8, 16, 2, 2)
    assert need >= 100 * 16 * 2                                   # the pre-activation's gradient
    assert _backward(lib, rows=100, n=16, act=2, ws=None, ws_bytes=0) == 8
    assert _backward(lib, rows=100, n=16, act=2, ws_bytes=need - 1) == 8
    assert _backward(lib, rows=100, n=16, act=2, ws=ctypes.c_void_p(264), ws_bytes=need) == 9
    assert lib.fda_linear_backward_workspace_bytes(1, 100, 1, 0, 16, 2, 2) == 0


def test_python_refusals():
    x, w = torch.zeros(3, 4), torch.zeros(2, 4)
    with pytest.raises(ValueError, match="activation must be one of"):
        ops3d_b200.fused_linear(x, w, activation="swish")
    with pytest.raises(ValueError, match="activation must be one of"):
        ops3d_b200.fused_linear(x, w, activation=None)
    with pytest.raises(ValueError, match="group_start_index is required"):
        ops3d_b200.grouped_linear(x, w[None], None)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        ops3d_b200.fused_linear(x, w)
    with pytest.raises(ValueError, match="goes with n_groups"):
        ops3d_b200.FeedForward(4, 8)(x, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="goes with n_groups"):
        ops3d_b200.FeedForward(4, 8, n_groups=2)(x)
    with pytest.raises(ValueError, match="activation must be one of"):
        ops3d_b200.FeedForward(4, 8, activation="tanh")


class Binding:
    """y = (sum of x) everywhere; counts the calls of the node entry point."""
    nodes = 0

    def linear(self, x, weight, bias, residual, starts, activation):
        self.nodes += 1
        with torch.no_grad(), torch._C._DisableTorchDispatch():
            return torch.full((*x.shape[:-1], weight.shape[-2]), float(x.detach().double().sum()))

    def linear_forward(self, x, weight, bias, residual, starts, activation):
        return x.sum() * torch.ones(*x.shape[:-1], weight.shape[-2])

    def linear_backward(self, x, weight, bias, starts, grad, activation, need_x, need_weight, need_bias):
        return (grad.sum() * torch.ones_like(x) if need_x else None, torch.zeros_like(weight) if need_weight else None,
                torch.zeros_like(bias) if need_bias else None)


@pytest.fixture
def binding(monkeypatch):
    fake = Binding()
    monkeypatch.setattr(linear_mod, "_C", fake)
    return fake


def test_plain_calls_take_the_node_and_other_modes_the_function(binding):
    x, w, b = torch.rand(3, 4), torch.rand(2, 4, requires_grad=True), torch.rand(2)
    ops3d_b200.fused_linear(x, w, b)
    assert binding.nodes == 1
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="jvp"):
            ops3d_b200.fused_linear(forward_ad.make_dual(x, torch.ones_like(x)), w, b)
    wd = w.detach()
    traced = torch.jit.trace(lambda v: ops3d_b200.fused_linear(v, wd, b), (x,), check_trace=False)
    assert binding.nodes == 1
    assert torch.allclose(traced(x + 1), ops3d_b200.fused_linear(x + 1, wd, b)) and not torch.allclose(traced(x + 1), traced(x))

    class Mine(ops3d_b200.FusedLinearFunction):
        pass

    r = torch.rand(3, 2, requires_grad=True)
    xg = x.clone().requires_grad_(True)
    y = Mine.apply(xg, w, b, r)
    gx, gr = torch.autograd.grad(y, (xg, r), torch.full((3, 2), 2.0))
    assert torch.equal(gx, torch.full_like(x, 12.0)) and torch.equal(gr, torch.full((3, 2), 2.0))


def test_layer_keeps_its_parameters():
    from ops3d_b200.msda3d import MSDeformAttn3D

    plain = MSDeformAttn3D(32, 2, 4, 4)
    assert set(plain.state_dict()) == {f"{m}.{p}" for m in ("sampling_offsets", "attention_weights", "value_proj", "output_proj")
                                       for p in ("weight", "bias")}
    assert plain.value_proj.weight.shape == (32, 32)
    levels = MSDeformAttn3D(32, 2, 4, 4, level_value_proj=True)
    assert levels.value_proj.weight.shape == (2, 32, 32) and levels.value_proj.bias.shape == (2, 32)
    assert set(levels.state_dict()) == set(plain.state_dict())


def test_a_layer_pickled_before_the_level_projections_has_one_for_all():
    from ops3d_b200.msda3d import MSDeformAttn3D

    layer = MSDeformAttn3D(32, 2, 4, 4)
    del layer.__dict__["level_value_proj"]
    assert layer.level_value_proj is False
    assert MSDeformAttn3D(32, 2, 4, 4, level_value_proj=True).level_value_proj is True


def test_a_residual_of_another_type_keeps_its_bits():
    from ops3d_b200.linear import add_residual

    y, r = torch.ones(3, 4, dtype=torch.bfloat16), torch.rand(3, 4)
    assert add_residual(y, r).dtype == torch.float32 and torch.equal(add_residual(y, r), r + 1)
    with pytest.raises(RuntimeError, match="shape of the output"):
        add_residual(y, r[:1])


def test_waits_that_ran_out_are_counted_in_python(binding, monkeypatch):
    monkeypatch.setattr(binding, "linear_timeouts", lambda: 3, raising=False)
    assert ops3d_b200.linear_timeouts() == 3
    monkeypatch.undo()
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="linear_timeouts"):
            ops3d_b200.linear_timeouts()
