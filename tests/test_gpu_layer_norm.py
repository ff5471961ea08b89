"""``layer_norm`` against the formulas in 64 bits.

Tolerances, per element, with u = 2^-24 (half a step of fp32) and D the most additions an element passes on its way into a sum over a row:
16 values of a thread, 5 steps over a warp, 16 warps, or (width / 512 of a thread in rows too wide for registers).

* s = x + r: u |s|;  mean: (D + 1) u mean|s|;  d = s - mean: both, and u |d|            (e_d)
* var: 2 mean(|d| e_d) + (D + 2) u var;  q = 1 / sqrt(var + eps): half of that relative to var + eps, and 2 u   (r_q)
* y: |w| q (e_d + |d| (r_q + 3 u)) + u (|y| + |b|)
* the gradients the same way, term by term; sums over rows are off by (rows + 2) u of the sum of their magnitudes
* a rounding to the output's type: half a step
"""
import threading

import pytest
import torch

from ops3d_b200 import LayerNorm, LayerNormFunction, layer_norm

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24
MORE = 1.02  # second-order terms of the bounds


def rounding(v, dtype):
    fi = torch.finfo(dtype)
    return (v.abs() * (fi.eps / 2) * (1 + fi.eps) + fi.tiny * fi.eps / 2) * MORE


def reference(x, w, b, r, eps, dy=None, dsum=None):
    """{name: (value, bound)} in 64 bits, before the outputs' roundings."""
    C = x.shape[-1]
    x, w, b, r, dy, dsum = (None if t is None else t.detach().double() for t in (x, w, b, r, dy, dsum))
    x = x.reshape(-1, C)
    rows, D = x.shape[0], max(40, C / 512 + 24)
    w = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w
    b = torch.zeros(C, dtype=torch.float64, device=x.device) if b is None else b
    s = x if r is None else x + r.reshape(-1, C)

    def mean(t):
        return t.mean(-1, keepdim=True)

    mu = mean(s)
    d = s - mu
    ed = (0 if r is None else U * s.abs()) + (D + 1) * U * mean(s.abs()) + U * d.abs()
    var = mean(d * d)
    var_err = 2 * mean(d.abs() * ed) + mean(ed * ed) + (D + 2) * U * var
    q = 1 / torch.sqrt(var + eps)
    rq = 0.5 * var_err / (var + eps) + 2 * U
    z = d * q
    y = z * w + b
    out = dict(y=(y, w.abs() * q * (ed + d.abs() * (rq + 3 * U)) + U * (y.abs() + b.abs())), s=(s, U * s.abs()))
    if dy is None:
        return out
    dy = dy.reshape(-1, C)
    g = dy * w
    level, A = mean(g), mean(g * d)
    level_err = (D + 2) * U * mean(g.abs())
    A_err = mean(g.abs() * ed) + (D + 3) * U * mean((g * d).abs())
    along = q * q * A
    along_err = q * q * (A_err + A.abs() * (2 * rq + 4 * U))
    ds = q * (g - level - d * along)
    ds_err = q * (2 * U * g.abs() + level_err + d.abs() * along_err + ed * along.abs() + 4 * U * (g.abs() + level.abs() + (d * along).abs())) \
        + ds.abs() * (rq + 2 * U)
    if dsum is not None:
        ds = ds + dsum.reshape(-1, C)
        ds_err = ds_err + U * ds.abs()
    z_err = q * (ed + d.abs() * (rq + 2 * U))
    out.update(ds=(ds, ds_err), weight=((dy * z).sum(0), (dy.abs() * z_err).sum(0) + (rows + 2) * U * (dy * z).abs().sum(0)),
               bias=(dy.sum(0), (rows + 2) * U * dy.abs().sum(0)))
    return out


def compare(got, want, name):
    value, bound = want
    value, bound = value.reshape(got.shape), bound.reshape(got.shape) * MORE + rounding(value, got.dtype).reshape(got.shape)
    assert torch.isfinite(got).all(), name
    worst = ((got.detach().double() - value).abs() / bound.clamp_min(1e-300)).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3f} of the bound"


def make(shape, dtype, params=None, residual=None, seed=0, scale=1.0, mean=0.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*size, dt=dtype, scale=1.0, mean=0.0):
        return (torch.randn(*size, generator=gen, device=DEV) * scale + mean).to(dt)

    C = shape[-1]
    x = normal(*shape, scale=scale, mean=mean)
    w, b = (normal(C, dt=params or dtype, scale=0.3, mean=1.0), normal(C, dt=params or dtype, scale=0.3)) if params is not False else (None, None)
    r = None if residual is None else normal(*shape, dt=residual, scale=2.0, mean=0.3)
    return x, w, b, r, normal(*shape), None if r is None else normal(*shape, dt=residual)


def check(x, w, b, r, dy, dsum=None, eps=1e-5):
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b, r)]
    keep = dsum is not None
    out = layer_norm(*leaves[:3], residual=leaves[3], eps=eps, return_sum=keep)
    y, s = out if keep else (out, None)
    want = reference(x, w, b, r, eps, dy, dsum)
    assert y.dtype == x.dtype and y.shape == x.shape
    compare(y, want["y"], "y")
    if keep:
        assert s.dtype == r.dtype
        compare(s, want["s"], "s")
    names = [n for n, t in zip(("x", "weight", "bias", "residual"), leaves) if t is not None]
    used = [t for t in leaves if t is not None]
    grads = dict(zip(names, torch.autograd.grad([y, s] if keep else [y], used, [dy, dsum] if keep else [dy])))
    for name, g in grads.items():
        leaf = dict(zip(names, used))[name]
        assert g.dtype == leaf.dtype and g.shape == leaf.shape
        compare(g, want["ds" if name in ("x", "residual") else name], "grad_" + name)


WIDTHS = [1, 2, 7, 8, 9, 31, 32, 33, 57, 64, 65, 99, 127, 128, 129, 255, 256, 257, 259, 264, 505, 512, 513, 520, 1000, 1024, 1031, 2048, 4096,
          4100, 8176, 8177, 8192, 8193, 20001]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_widths(width, dtype):
    for i, rows in enumerate((1, 3, 17)):
        params = [dtype, F32, False][(i + width) % 3]
        residual = [None, dtype, F32][(i + width // 3) % 3]
        x, w, b, r, dy, dsum = make((rows, width), dtype, params, residual, seed=width + i)
        check(x, w, b, r, dy, dsum if (width + i) % 2 else None)


@pytest.mark.parametrize("rows,width,dtype,residual", [(40000, 64, BF16, BF16), (20001, 259, BF16, None), (9001, 250, F16, F32), (5003, 131, F32, F32),
                                                       (5000, 512, F16, F16), (4001, 1024, BF16, F32), (2001, 1030, F16, F16),
                                                       (1501, 4099, F32, None), (40001, 8, F16, None), (40001, 3, F32, F32),
                                                       (700, 9001, BF16, BF16)])
def test_teams_take_many_rows(rows, width, dtype, residual):
    x, w, b, r, dy, dsum = make((rows, width), dtype, F32, residual, seed=rows)
    check(x, w, b, r, dy, dsum)


@pytest.mark.parametrize("width", [256, 259, 1030, 9000])
def test_a_mean_far_from_zero(width):
    """No cancellation: deviations of 1 around 1000 are as exact as fp32 holds them."""
    x, w, b, r, dy, _ = make((64, width), F32, None, None, mean=1000.0)
    check(x, w, b, r, dy)
    y = layer_norm(torch.full((3, width), 7.25, device=DEV), eps=1e-5)
    assert (y.abs() <= 40 * U * 7.25 * 1e-5 ** -0.5 * MORE).all()     # deviations of a constant row are the mean's error


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_eps_and_shapes(dtype):
    for shape, eps in (((5, 40), 0.5), ((2, 3, 4, 24), 1e-12), ((77,), 1e-3)):
        x, w, b, r, dy, dsum = make(shape, dtype, F32, dtype, seed=len(shape))
        check(x, w, b, r, dy, dsum, eps=eps)


def test_no_rows():
    w = torch.ones(24, device=DEV, requires_grad=True)
    x = torch.zeros(0, 24, device=DEV, requires_grad=True)
    y = layer_norm(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), torch.zeros(0, 24, device=DEV))
    assert y.shape == gx.shape == (0, 24) and torch.equal(gw, torch.zeros_like(w))


@pytest.mark.parametrize("width", [64, 99, 259, 600])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_strides_and_bases(width, dtype):
    """Transposed, sliced, broadcast and misaligned operands give what contiguous copies give."""
    x, w, b, r, dy, _ = make((width, 33), dtype, F32, dtype)
    x, r, dy = x.t(), r.t(), dy.t()                                          # [33, width]
    w, b = make((width,), F32)[0], make((2 * width,), F32, seed=1)[0][::2]   # every other number
    base = torch.zeros(33 * width + 1, dtype=dtype, device=DEV)
    odd = base[1:].view(33, width)
    odd.copy_(x)
    line = dy[:1].expand(33, width)
    for a, g in ((x, dy), (odd, line)):
        leaves = [t.detach().requires_grad_(True) for t in (a, w, b, r)]
        same = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True) for t in (a, w, b, r)]
        ys, yc = (layer_norm(v[0], v[1], v[2], residual=v[3]) for v in (leaves, same))
        assert torch.equal(ys, yc)
        for p, q in zip(torch.autograd.grad(ys, leaves, g), torch.autograd.grad(yc, same, g.contiguous())):
            assert torch.equal(p, q)
    check(x, w, b, r, dy)
    few = torch.randn(1, width, device=DEV).to(dtype).requires_grad_(True)   # a broadcast input's gradient is the sum over its copies
    full = few.detach().expand(33, width).contiguous().requires_grad_(True)
    (gf,) = torch.autograd.grad(layer_norm(few.expand(33, width), w, b), few, dy)
    (gx,) = torch.autograd.grad(layer_norm(full, w, b), full, dy)
    assert torch.equal(gf, gx.sum(0, keepdim=True))


@pytest.mark.parametrize("width", [8, 64, 259, 512, 1030, 9001])
def test_rows_do_not_see_their_neighbours(width):
    """A row of NaN or infinity leaves the others as they are, vectors that two rows share among them."""
    x, w, b, r, dy, dsum = make((40, width), BF16, F32, BF16)
    clean = [t.detach().clone().requires_grad_(True) for t in (x, r)]
    y = layer_norm(clean[0], w, b, residual=clean[1])
    gx = torch.autograd.grad(y, clean[0], dy)[0]
    bad = (0, 7, 13, 39)
    x2 = x.clone()
    for row, value in zip(bad, (float("nan"), float("inf"), -float("inf"), float("nan"))):
        x2[row, -1] = value
        x2[row, 0] = value
    leaf = x2.requires_grad_(True)
    y2 = layer_norm(leaf, w, b, residual=r)
    gx2 = torch.autograd.grad(y2, leaf, dy)[0]
    good = [i for i in range(40) if i not in bad]
    assert torch.equal(y2[good], y[good]) and torch.equal(gx2[good], gx[good])
    assert y2[list(bad)].isnan().all() and gx2[list(bad)].isnan().all()


def test_only_the_wanted_gradients():
    x, w, b, r, dy, dsum = make((50, 99), F16, F32, F32)
    full = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
    want = torch.autograd.grad(layer_norm(*full[:3], residual=full[3]), full, dy)
    for i in range(4):
        leaves = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, w, b, r))]
        (got,) = torch.autograd.grad(layer_norm(*leaves[:3], residual=leaves[3]), leaves[i], dy)
        assert torch.equal(got, want[i])


def test_either_output_alone_has_gradients():
    x, w, b, r, dy, dsum = make((50, 99), F32, F32, F32)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
    y, s = layer_norm(*leaves[:3], residual=leaves[3], return_sum=True)
    gx, gr = torch.autograd.grad(s, (leaves[0], leaves[3]), dsum, retain_graph=True)
    assert torch.equal(gx, dsum) and torch.equal(gr, dsum)                   # nothing comes through the norm
    gx, gw = torch.autograd.grad(y, leaves[:2], dy)
    want = reference(x, w, b, r, 1e-5, dy)
    compare(gx, want["ds"], "x")
    compare(gw, want["weight"], "weight")


def test_gradients_against_differences():
    """The formula's gradients along a direction, against central differences of the definition in 64 bits; what the differences
    themselves are off by is estimated from two distances."""
    x, w, b, r, dy, _ = make((9, 37), F32, F32, F32)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
    grads = torch.autograd.grad(layer_norm(*leaves[:3], residual=leaves[3]), leaves, dy)
    bounds = reference(x, w, b, r, 1e-5, dy)
    for i, name in enumerate(("ds", "weight", "bias", "ds")):
        v = torch.randn(leaves[i].shape, dtype=torch.float64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(i))

        def quotient(h):
            total = 0
            for sign in (1, -1):
                moved = [t.detach().double() + (sign * h * v if j == i else 0) for j, t in enumerate(leaves)]
                total = total + sign * (reference(*moved, 1e-5)["y"][0] * dy.double()).sum()
            return (total / (2 * h)).item()

        near, far = quotient(2.0 ** -12), quotient(2.0 ** -11)
        got = (grads[i].double() * v).sum().item()
        value, bound = bounds[name]
        slack = ((bound * MORE + rounding(value, F32)).reshape(v.shape) * v.abs()).sum().item()
        assert abs(got - near) <= slack + abs(near - far) + 1e-9 * abs(near)


def test_repeated_calls_are_equal():
    x, w, b, r, dy, dsum = make((30001, 259), BF16, F32, F32)
    results = []
    for _ in range(3):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
        y, s = layer_norm(*leaves[:3], residual=leaves[3], return_sum=True)
        results.append([y, s, *torch.autograd.grad([y, s], leaves, [dy, dsum])])
    for other in results[1:]:
        assert all(torch.equal(a, c) for a, c in zip(results[0], other))


def test_the_function_is_the_node():
    class Mine(LayerNormFunction):
        pass

    x, w, b, r, dy, dsum = make((50, 99), BF16, F32, F32)
    out = []
    for apply in (LayerNormFunction.apply, Mine.apply):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
        y, s = apply(*leaves, 1e-5, True)
        grads = torch.autograd.grad([y, s], leaves, [dy, dsum], retain_graph=True)
        (only,) = torch.autograd.grad(s, leaves[0], dsum)
        out.append([y, s, *grads, only])
        assert torch.equal(only, dsum.to(BF16))
    assert all(torch.equal(a, c) for a, c in zip(*out))


def test_layer_and_state():
    torch.manual_seed(0)
    theirs = torch.nn.LayerNorm(96).to(DEV)
    torch.nn.init.normal_(theirs.weight)
    torch.nn.init.normal_(theirs.bias)
    mine = LayerNorm(96).to(DEV)
    mine.load_state_dict(theirs.state_dict())
    x = torch.randn(7, 5, 96, device=DEV)
    compare(mine(x), reference(x, theirs.weight, theirs.bias, None, 1e-5)["y"], "y")
    half = x.to(BF16)
    y, s = mine(half, residual=x, return_sum=True)
    assert y.dtype == BF16 and s.dtype == F32 and torch.equal(s, half.float() + x)
    with torch.autocast("cuda", dtype=F16):
        assert mine(half).dtype == BF16
    assert LayerNorm(96, bias=False).bias is None


def test_captured_pass_follows_its_inputs():
    x, w, b, r, dy, dsum = make((301, 259), BF16, F32, BF16)
    stream = torch.cuda.Stream()
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b, r)]

    def run():
        y, s = layer_norm(*leaves[:3], residual=leaves[3], return_sum=True)
        return [y, s, *torch.autograd.grad([y, s], leaves, [dy, dsum])]

    with torch.cuda.stream(stream):
        for _ in range(2):
            run()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = run()
    for seed in (1, 2):
        new = make((301, 259), BF16, F32, BF16, seed=seed)
        with torch.no_grad():
            for leaf, value in zip(leaves, new[:4]):
                leaf.copy_(value)
            dy.copy_(new[4])
            dsum.copy_(new[5])
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, run()):
            assert torch.equal(a, c)


def test_streams_and_threads():
    """Calls at once, each on a stream of its own."""
    cases = [make((2001 + i, 259 - i), BF16, F32, BF16, seed=i) for i in range(4)]

    def run(case):
        leaves = [t.detach().requires_grad_(True) for t in case[:4]]
        y = layer_norm(*leaves[:3], residual=leaves[3])
        return [y, *torch.autograd.grad(y, leaves, case[4])]

    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i] = run(cases[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for a, c in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, c))


def test_more_than_2_31_elements():
    """Offsets beyond 32 bits: the last rows of a tensor of 2^31 elements and more."""
    rows, width = (1 << 23) + 5, 259
    x = torch.zeros(rows, width, dtype=BF16, device=DEV)
    x[-70:] = make((70, width), BF16)[0]
    x.requires_grad_(True)
    y = layer_norm(x)
    dy = torch.zeros_like(y)
    dy[-70:] = make((70, width), BF16, seed=1)[0]
    (gx,) = torch.autograd.grad(y, x, dy)
    want = reference(x[-70:], None, None, None, 1e-5, dy[-70:])
    compare(y[-70:], want["y"], "y")
    compare(gx[-70:], want["ds"], "x")
    assert not y[:100].any() and not gx[:100].any()
