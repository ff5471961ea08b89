"""Host side of layer norm, routing and the rows sorted by expert: what the C ABI and the Python entry points refuse before a kernel is
launched, workspaces, modules, and what has to see the autograd Functions.  No device needed."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import ops3d_b200
import ops3d_b200.experts as experts_mod
import ops3d_b200.norm as norm_mod
from ops3d_b200 import capi

P, ODD = ctypes.c_void_p(256), ctypes.c_void_p(264)
F32, F16, BF16 = 0, 1, 2


def _norm(lib, x=P, w=P, b=P, r=P, y=P, s=None, rows=4, width=8, eps=1e-5, dt=BF16, pdt=F32, rdt=F32):
    return lib.fda_layer_norm_forward(x, w, b, r, y, s, rows, width, eps, dt, pdt, rdt, None)


def _norm_backward(lib, x=P, r=P, dy=P, ds=None, dx=P, dr=None, dw=P, ws=P, ws_bytes=1 << 40, rows=4, width=8, dt=BF16, pdt=F32, rdt=F32):
    return lib.fda_layer_norm_backward(x, P, r, dy, ds, dx, dr, dw, None, ws, ws_bytes, rows, width, 1e-5, dt, pdt, rdt, None)


def test_layer_norm_arguments():
    lib = capi.load()
    for call in (_norm, _norm_backward):
        assert call(lib, dt=3) == 2 and call(lib, dt=-1) == 2
        assert call(lib, dt=BF16, pdt=F16) == 2 and call(lib, dt=F32, pdt=BF16) == 2
        assert call(lib, dt=BF16, rdt=F16) == 2 and call(lib, dt=F32, rdt=F16) == 2
        assert call(lib, width=0) == 6 and call(lib, rows=-1) == 6 and call(lib, rows=1 << 31) == 6 and call(lib, width=1 << 26) == 6
        assert call(lib, x=None) == 1 and call(lib, x=ODD) == 9 and call(lib, r=ODD) == 9
    assert _norm(lib, y=None) == 1 and _norm(lib, r=None, s=P) == 1 and _norm(lib, y=ODD) == 9 and _norm(lib, s=ODD) == 9
    assert _norm(lib, rows=0, x=None) == 0
    assert _norm_backward(lib, dy=None) == 1 and _norm_backward(lib, r=None, ds=P) == 1 and _norm_backward(lib, r=None, dr=P) == 1
    assert _norm_backward(lib, dy=ODD) == 9 and _norm_backward(lib, ds=ODD) == 9 and _norm_backward(lib, dx=ODD) == 9 and _norm_backward(lib, dr=ODD) == 9
    need = lib.fda_layer_norm_backward_workspace_bytes(4, 8, BF16)
    assert need >= 2 * 8 * 4
    assert _norm_backward(lib, ws=None) == 8 and _norm_backward(lib, ws_bytes=need - 1) == 8 and _norm_backward(lib, ws=ODD) == 9
    assert lib.fda_layer_norm_backward_workspace_bytes(0, 8, BF16) == 0 and lib.fda_layer_norm_backward_workspace_bytes(4, 0, BF16) == 0
    # partial sums of blocks: bounded by the device, not by the rows
    assert lib.fda_layer_norm_backward_workspace_bytes(1 << 30, 256, BF16) < 64 << 20


def _route(lib, ptr=P, bias=None, tokens=4, experts=8, k=2, score=0, groups=1, top=1, gscore=0, dt=F32):
    return lib.fda_route_forward(ptr, bias, ptr, ptr, tokens, experts, k, score, groups, top, gscore, 1, 1.0, dt, None)


def test_route_arguments():
    lib = capi.load()
    assert _route(lib, dt=3) == 2
    assert _route(lib, tokens=-1) == 6 and _route(lib, tokens=1 << 31) == 6 and _route(lib, experts=0) == 6 and _route(lib, k=0) == 6
    assert _route(lib, k=9) == 6 and _route(lib, groups=3) == 6 and _route(lib, groups=4, top=5) == 6 and _route(lib, groups=4, top=0) == 6
    assert _route(lib, groups=4, top=1, k=3) == 6                 # two candidates
    assert _route(lib, experts=1025) == 11 and _route(lib, experts=66, k=33) == 11 and _route(lib, experts=66, groups=33, top=33) == 11
    assert _route(lib, score=2) == 13 and _route(lib, score=-1) == 13 and _route(lib, gscore=2) == 13
    assert lib.fda_status_string(13) not in (b"ok", b"unknown status")
    assert _route(lib, ptr=None) == 1 and _route(lib, tokens=0, ptr=None) == 0
    back = lib.fda_route_backward
    assert back(P, P, P, P, 4, 8, 9, 0, 1, 1.0, F32, None) == 6 and back(P, P, P, P, 4, 8, 2, 0, 1, 1.0, 7, None) == 2
    assert back(P, None, P, P, 4, 8, 2, 0, 1, 1.0, F32, None) == 1 and back(None, None, None, None, 0, 8, 2, 0, 1, 1.0, F32, None) == 0


def _dispatch(lib, x=P, e=P, rows=P, starts=P, pos=P, ws=P, ws_bytes=1 << 40, tokens=4, k=2, experts=8, width=8, dt=BF16):
    return lib.fda_dispatch_rows(x, e, rows, starts, pos, ws, ws_bytes, tokens, k, experts, width, dt, None)


def test_row_arguments():
    lib = capi.load()
    assert _dispatch(lib, dt=3) == 2 and _dispatch(lib, tokens=-1) == 6 and _dispatch(lib, k=0) == 6 and _dispatch(lib, width=0) == 6
    assert _dispatch(lib, width=1 << 26) == 6 and _dispatch(lib, tokens=1 << 30, k=2) == 6 and _dispatch(lib, experts=0) == 6
    assert _dispatch(lib, k=33) == 11 and _dispatch(lib, experts=1025) == 11
    assert all(_dispatch(lib, **{n: None}) == 1 for n in ("x", "e", "rows", "starts", "pos"))
    assert lib.fda_dispatch_workspace_bytes(4, 2, 8) == 0         # few entries are counted where they are placed
    need = lib.fda_dispatch_workspace_bytes(40000, 2, 8)
    assert need > 0 and _dispatch(lib, tokens=400000, ws=None) == 8 and _dispatch(lib, tokens=40000, ws_bytes=need - 1) == 8
    assert _dispatch(lib, tokens=400000, ws=ODD) == 9
    assert lib.fda_dispatch_workspace_bytes(1 << 29, 2, 1024) < 4 << 20
    assert _dispatch(lib, x=ODD) == 9 and _dispatch(lib, rows=ODD) == 9
    assert lib.fda_dispatch_workspace_bytes(0, 2, 8) == 0 and lib.fda_dispatch_workspace_bytes(4, 2, 1025) == 0
    comb = lambda rows=P, pos=P, w=P, r=P, y=P, t=4, k=2, c=8, dt=BF16, wdt=F32: lib.fda_combine_rows(rows, pos, w, r, y, t, k, c, dt, wdt, None)  # noqa: E731
    assert comb(dt=3) == 2 and comb(wdt=3) == 2 and comb(t=-1) == 6 and comb(k=33) == 11 and comb(rows=None) == 1 and comb(pos=None) == 1
    assert comb(rows=ODD) == 9 and comb(r=ODD) == 9 and comb(y=ODD) == 9 and comb(t=0, rows=None) == 0
    need = lib.fda_combine_rows_backward_workspace_bytes(4, 2)
    assert need >= 32 and lib.fda_combine_rows_backward_workspace_bytes(0, 2) == 0 == lib.fda_combine_rows_backward_workspace_bytes(1 << 30, 2)
    back = lambda rows=P, pos=P, w=P, dy=P, dr=P, dw=P, ws=P, ws_bytes=need, t=4, dt=BF16, wdt=F32: lib.fda_combine_rows_backward(  # noqa: E731
        rows, pos, w, dy, dr, dw, ws, ws_bytes, t, 2, 8, dt, wdt, None)
    assert back(dt=3) == 2 and back(wdt=3) == 2 and back(rows=None) == 1 and back(pos=None) == 1 and back(dy=None) == 1
    assert back(ws=None) == 8 and back(ws_bytes=need - 1) == 8 and back(ws=ODD) == 9
    assert back(dr=ODD) == 9 and back(dy=ODD) == 9 and back(dr=None, dw=None, dy=None) == 0 and back(t=0) == 0


def test_python_refusals():
    x = torch.zeros(3, 4)
    e = torch.zeros(3, 2, dtype=torch.int64)
    for call in (lambda: ops3d_b200.layer_norm(x), lambda: ops3d_b200.route_experts(x, 2), lambda: ops3d_b200.dispatch_rows(x, e, 4),
                 lambda: ops3d_b200.combine_rows(torch.zeros(6, 4), (e, e))):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call()
    with pytest.raises(ValueError, match="return_sum needs a residual"):
        ops3d_b200.layer_norm(x, return_sum=True)
    for bad in ("relu", None, []):
        with pytest.raises(ValueError, match="score must be one of softmax, sigmoid"):
            ops3d_b200.route_experts(x, 2, score=bad)
        with pytest.raises(ValueError, match="group_score must be one of max, top2"):
            ops3d_b200.route_experts(x, 2, group_score=bad)
    for bad in (dict(n_groups=3), dict(n_groups=4, top_groups=5), dict(top_k=9), dict(n_groups=4, top_groups=1, top_k=3)):
        with pytest.raises(ValueError, match="n_groups must divide"):
            ops3d_b200.ExpertFeedForward(8, 16, 8, **bad)
    with pytest.raises(ValueError, match="score must be one of"):
        ops3d_b200.ExpertFeedForward(8, 16, 8, score="none")


class Binding:
    """Every output: the sum of the first argument everywhere; counts the calls of the node entry points."""
    nodes = 0

    def _first(self, t, shape):
        return t.sum() * torch.ones(shape)

    def _node(self, t, shape):
        self.nodes += 1
        with torch.no_grad(), torch._C._DisableTorchDispatch():
            return torch.full(shape, float(t.detach().double().sum()))

    def layer_norm(self, x, w, b, r, eps, keep):
        return [self._node(x, x.shape), None]

    def layer_norm_forward(self, x, w, b, r, eps, keep):
        return [self._first(x, x.shape), None]

    def layer_norm_backward(self, x, w, b, r, grad, grad_sum, eps, *need):
        return [grad.sum() * torch.ones_like(x), None, None, None]

    def route(self, logits, bias, k, *options):
        return [self._node(logits, (*logits.shape[:-1], k)), torch.zeros(*logits.shape[:-1], k, dtype=torch.int64)]

    def route_forward(self, logits, bias, k, *options):
        return [self._first(logits, (*logits.shape[:-1], k)), torch.zeros(*logits.shape[:-1], k, dtype=torch.int64)]

    def route_backward(self, logits, experts, grad, *options):
        assert len(options) == 3
        return grad.sum() * torch.ones_like(logits)

    def _order(self, experts, n):
        return torch.zeros(n + 1, dtype=torch.int64), torch.zeros_like(experts)

    def dispatch(self, x, experts, n):
        return [self._node(x, (experts.numel(), x.shape[-1])), *self._order(experts, n)]

    def dispatch_forward(self, x, experts, n):
        return [self._first(x, (experts.numel(), x.shape[-1])), *self._order(experts, n)]

    def combine(self, rows, position, weights, residual):
        return self._node(rows, (*position.shape[:-1], rows.shape[-1]))

    def combine_forward(self, rows, position, weights, residual):
        return rows.sum() * torch.ones(*position.shape[:-1], rows.shape[-1])

    def combine_backward(self, rows, position, weights, grad, need_rows, need_weights):
        return [grad.sum() * torch.ones(position.numel(), grad.shape[-1]) if need_rows else None, None]


@pytest.fixture
def binding(monkeypatch):
    fake = Binding()
    for mod in (norm_mod, experts_mod):
        monkeypatch.setattr(mod, "_C", fake)
    return fake


EXPERTS = torch.zeros(3, 2, dtype=torch.int64)
OPS = {
    "norm": (norm_mod.LayerNormFunction, torch.rand(3, 4), lambda f, v: f(v, None, None, None, 1e-5, False)[0]),
    "route": (experts_mod.RouteExpertsFunction, torch.rand(3, 4), lambda f, v: f(v, None, 2, 0, 1, 1, 0, True, 1.0)[0]),
    "dispatch": (experts_mod.DispatchRowsFunction, torch.rand(3, 4), lambda f, v: f(v, EXPERTS, 4)[0]),
    "combine": (experts_mod.CombineRowsFunction, torch.rand(6, 4), lambda f, v: f(v, EXPERTS, None, None)),
}


@pytest.mark.parametrize("op", OPS)
def test_plain_calls_take_the_node_and_other_modes_the_function(op, binding):
    function, x, call = OPS[op]
    x = x.clone()
    call(function.apply, x)
    assert binding.nodes == 1
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="jvp"):
            call(function.apply, forward_ad.make_dual(x, torch.ones_like(x)))
    traced = torch.jit.trace(lambda v: call(function.apply, v), (x,), check_trace=False)
    assert binding.nodes == 1
    assert torch.allclose(traced(x + 1), call(function.apply, x + 1)) and not torch.allclose(traced(x + 1), traced(x))

    class Mine(function):
        pass

    leaf = x.clone().requires_grad_(True)
    out = call(Mine.apply, leaf)
    (grad,) = torch.autograd.grad(out.sum(), leaf)
    assert torch.equal(grad, torch.full_like(x, out.numel()))


def test_module_state():
    assert set(ops3d_b200.LayerNorm(8).state_dict()) == {"weight", "bias"}
    block = ops3d_b200.ExpertFeedForward(8, 16, 4, balanced=True)
    assert set(block.state_dict()) == {"norm.weight", "norm.bias", "router", "balance", *(f"experts.{p}{i}" for p in ("weight", "bias") for i in (1, 2))}
    assert block.router.shape == (4, 8) and block.experts.weight1.shape == (4, 16, 8)
    assert "balance" not in ops3d_b200.ExpertFeedForward(8, 16, 4, norm=False).state_dict()
