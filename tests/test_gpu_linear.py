"""Linear operators (``fused_linear``, ``grouped_linear``) against the formulas in 64 bits.

Tolerances, from the arithmetic alone (``eps`` of the tensors' type, all quantities per element):

* a rounding to the type is off by ``eps / 2`` of the value, below the normal range by half the smallest step;
* a sum of n products in fp32 is off by at most ``n * 2^-23`` of the sum of their magnitudes, whatever its order and whether an
  addition rounds or truncates;
* act and act' are evaluated in fp32, off by less than ``2^-20 * (1 + |v|)``; their slopes are at most 1.13, so an error of the
  pre-activation passes on at most 1.13 times as large;
* for 16-bit types with an activation g is rounded to the type between the products.
"""
import math
import threading

import pytest
import torch

from ops3d_b200 import FeedForward, GroupedLinear, capi, fused_linear, grouped_linear

pytestmark = pytest.mark.gpu

DEV = "cuda"
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    assert capi.load().fda_linear_timeouts() == 0


def act64(v, act):
    c = math.sqrt(2 / math.pi)
    if act == "none":
        return v, torch.ones_like(v)
    if act == "relu":
        return v.clamp_min(0), (v > 0).double()
    if act == "gelu":
        cdf = torch.special.ndtr(v)
        return v * cdf, cdf + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        t = torch.tanh(c * (v + 0.044715 * v ** 3))
        return v * (1 + t) / 2, (1 + t) / 2 + v * (1 - t * t) * c * (1 + 3 * 0.044715 * v * v) / 2
    s = torch.sigmoid(v)
    return v * s, s * (1 + v * (1 - s))


def rounding(v, dtype):
    fi = torch.finfo(dtype)
    return v.abs() * (fi.eps / 2) * (1 + fi.eps) + fi.tiny * fi.eps / 2


def group_of_rows(starts, groups, rows):
    """Group of each row (-1: of none), from the documented rule."""
    s = [min(max(int(v), 0), rows) for v in starts]
    for i in range(1, len(s)):
        s[i] = max(s[i], s[i - 1])
    ends = s[1:] + ([rows] if len(s) == groups else [])
    out = torch.full((rows,), -1, dtype=torch.int64)
    for e in range(groups):
        out[s[e]:ends[e]] = e
    return out


def reference(x, w, b, r, dy, act, owner=None):
    """Values and bounds in 64 bits: y, dx, dW, db, each (value, bound).  w [E, N, K]; owner [rows of x] on the device."""
    dtype = x.dtype
    K, N = x.shape[-1], w.shape[-2]
    x2, dy2 = x.detach().double().reshape(-1, K), dy.detach().double().reshape(-1, N)
    r2 = None if r is None else r.detach().double().reshape(-1, N)
    w, b = w.detach().double(), None if b is None else b.detach().double()
    M, u23 = x2.shape[0], 2.0 ** -23
    y, ytol = torch.zeros(M, N, dtype=torch.float64, device=DEV), torch.zeros(M, N, dtype=torch.float64, device=DEV)
    dx, dxtol = torch.zeros_like(x2), torch.zeros_like(x2)
    dw, dwtol = torch.zeros_like(w), torch.zeros_like(w)
    db, dbtol = (torch.zeros(w.shape[:2], dtype=torch.float64, device=DEV) for _ in range(2))
    narrow = dtype != torch.float32 and act != "none"
    for e in range(w.shape[0]):
        rows = slice(None) if owner is None else (owner == e).nonzero()[:, 0]
        xe, ge = x2[rows], dy2[rows]
        if xe.shape[0] == 0:
            continue
        pre, mag = xe @ w[e].t(), xe.abs() @ w[e].abs().t()
        if b is not None:
            pre, mag = pre + b[e], mag + b[e].abs()
        preerr = (K + 2) * u23 * mag
        f, slope = act64(pre, act)
        evaluation = 0.0 if act in ("none", "relu") else 2.0 ** -20 * (1 + pre.abs())
        y[rows], ytol[rows] = f, 1.13 * preerr + evaluation
        g = ge * slope
        gerr = torch.zeros_like(g)
        if act != "none":
            gerr = ge.abs() * ((0 if act == "relu" else 1.13 * preerr) + evaluation)
        if narrow:
            gerr = gerr + rounding(g, dtype) * 1.01
        ga = g.abs() + gerr
        dx[rows], dxtol[rows] = g @ w[e], gerr @ w[e].abs() + (N + 2) * u23 * (ga @ w[e].abs())
        dw[e] = g.t() @ xe
        dwtol[e] = gerr.t() @ xe.abs() + (M + 2) * u23 * (ga.t() @ xe.abs())
        db[e], dbtol[e] = g.sum(0), gerr.sum(0) + (M + 2) * u23 * ga.sum(0)
    if r2 is not None:
        y, ytol = y + r2, ytol + 2 * u23 * (y.abs() + r2.abs())
    pairs = dict(y=(y, ytol), x=(dx, dxtol), weight=(dw, dwtol), bias=(db, dbtol))
    return {k: (v, t + rounding(v, dtype) * 1.01) for k, (v, t) in pairs.items()}


def compare(got, want, name):
    value, bound = want
    err = (got.detach().double().reshape(value.shape) - value).abs()
    assert torch.isfinite(got).all(), name
    worst = (err / bound.clamp_min(1e-300)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3f} of the bound, largest error {err.max().item():.3e}"


def make(lead, K, N, dtype, groups=None, bias=True, residual=True, seed=0, exact=False):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    g = () if groups is None else (groups,)

    def normal(*shape, scale=1.0):
        v = torch.randn(*shape, generator=gen, device=DEV) * scale
        return (v * 2).round().clamp(-4, 4).div(2).to(dtype) if exact else v.to(dtype)

    x, w = normal(*lead, K), normal(*g, N, K, scale=1.0 if exact else 1 / math.sqrt(K))
    return x, w, normal(*g, N) if bias else None, normal(*lead, N) if residual else None, normal(*lead, N)


def check(x, w, b, r, dy, act, starts=None):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b, r)]
    if starts is None:
        y = fused_linear(leaves[0], leaves[1], leaves[2], leaves[3], act)
        owner, w64, b64 = None, w[None], None if b is None else b[None]
    else:
        y = grouped_linear(leaves[0], leaves[1], starts, leaves[2], leaves[3], act)
        rows = x.shape[-2]
        owner = group_of_rows(starts.tolist(), w.shape[0], rows).repeat(x.shape[0] if x.dim() == 3 else 1).to(DEV)
        w64, b64 = w, b
    assert y.dtype == x.dtype and y.shape == (*x.shape[:-1], w.shape[-2])
    names = [n for n, t in zip(("x", "weight", "bias", "residual"), leaves) if t is not None]
    grads = dict(zip(names, torch.autograd.grad(y, [t for t in leaves if t is not None], dy)))
    want = reference(x, w64, b64, r, dy, act, owner)
    compare(y, want["y"], "y")
    for n in names:
        if n == "residual":
            assert torch.equal(grads[n], dy)
        else:
            assert grads[n].dtype == x.dtype and grads[n].shape == dict(x=x, weight=w, bias=b)[n].shape
            compare(grads[n], want[n], "grad_" + n)
    return y, grads


SIZES = [(1, 1, 1), (1, 256, 1024), (2, 8, 8), (5, 7, 9), (16, 64, 24), (17, 40, 200), (127, 64, 64), (128, 64, 256), (129, 72, 264),
         (300, 259, 250), (800, 256, 256), (1000, 1024, 96), (257, 16, 2048), (2049, 40, 513), (5000, 136, 128)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_sizes(size, dtype):
    M, K, N = size
    act = ACTS[(M + K + N) % 5]
    x, w, b, r, dy = make((M,), K, N, dtype, bias=(M + N) % 4 != 0, residual=K % 3 != 0, exact=act == "relu")
    check(x, w, b, r, dy, act)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_activations(act, dtype):
    """relu: inputs in halves, whose sums are exact, so that its derivative at 0 is met and decided."""
    for K, N in ((64, 136), (37, 50)):
        x, w, b, r, dy = make((3, 61), K, N, dtype, exact=act == "relu", seed=1)
        check(x, w, b, r, dy, act)
        check(x, w, None, None, dy, act)
    if act == "relu":
        assert (x.double() @ w.double().t() == 0).any()


@pytest.mark.parametrize("act", ACTS)
def test_far_values(act):
    """Pre-activations where exponentials over- and underflow."""
    v = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 5, -5, 9, -9, 30, -30, 90, -90, 200, -200, 1e4, -1e4], device=DEV)[:, None]
    one = torch.ones(1, 1, device=DEV)
    x = v.clone().requires_grad_(True)
    y = fused_linear(x, one, activation=act)
    (gx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    f, slope = act64(v.double(), act)
    # relative where the value is large; absolute below (the function's tail)
    assert ((y.double() - f).abs() <= 2e-6 * (1 + f.abs())).all()
    assert ((gx.double() - slope).abs() <= 4e-6).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_far_values_in_16_bits(act, dtype):
    """The same through the tensor-core kernels' paired functions, on every lane of a tile."""
    v = torch.cat([torch.linspace(-40, 40, 257), torch.tensor([0.0, -0.0, 1e-4, -1e-4, 90, -90, 200, -200, 6e4, -6e4])]).to(DEV)
    x = torch.zeros(v.numel(), 8, device=DEV)
    x[:, 3] = v
    x = x.to(dtype)
    w = torch.zeros(40, 8, device=DEV, dtype=dtype)
    w[:, 3] = 1
    dy = torch.ones(v.numel(), 40, device=DEV, dtype=dtype)
    leaf = x.clone().requires_grad_(True)
    y = fused_linear(leaf, w, activation=act)
    want = reference(x, w[None], None, None, dy, act)
    compare(y, want["y"], "y")
    (gx,) = torch.autograd.grad(y, leaf, dy)
    compare(gx, want["x"], "grad_x")
    assert torch.equal(y, y[:, :1].expand_as(y))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_infinities_do_not_depend_on_the_number_of_rows(act, dtype):
    """Plus and minus infinity and NaN as pre-activations: the same class of result for one row, few and many."""
    inf = float("inf")
    one = torch.ones(16, 1, device=DEV, dtype=dtype)
    results = []
    for rows in (3, 30, 300, 30000):
        x = torch.tensor([inf, -inf, float("nan")], device=DEV, dtype=dtype).repeat(rows // 3 + 1)[:rows, None].contiguous()
        y = fused_linear(x, one, activation=act)
        assert all(torch.equal(y[i::3].isnan(), y[i:i + 1].isnan().expand_as(y[i::3])) for i in range(3))
        results.append([float(y[i, 0]) for i in range(3)])
    for r in results:
        assert r[0] == inf and r[2] != r[2]
        assert (r[1] == results[0][1]) or (r[1] != r[1] and results[0][1] != results[0][1])
    if act in ("none", "relu", "gelu"):
        assert results[0][1] == {"none": -inf, "relu": 0.0, "gelu": 0.0}[act]


GROUPS = {
    "one": ([0], 1), "levels": ([0, 300, 375], 3), "ends": ([0, 100, 228, 400], 3), "empty": ([0, 0, 130, 130, 130, 390, 400], 7),
    "late": ([37, 166, 166], 3), "late-ends": ([5, 69, 133, 390], 3), "all-empty": ([9, 9, 9, 9], 3),
    "disorder": ([50, 20, 90, 70, 1000], 5), "outside": ([-7, 100, 1 << 40], 3), "singles": (list(range(0, 400, 9)), 45),
    "nothing": ([400, 400], 2),
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", GROUPS)
def test_groups(kind, dtype):
    starts, groups = GROUPS[kind]
    i = list(GROUPS).index(kind)
    act = ACTS[1:][i % 4] if i % 2 else "none"
    batch = (1, 2, 3)[i % 3]
    K, N = ((64, 72), (40, 264), (33, 29))[i % 3]
    x, w, b, r, dy = make((batch, 400) if batch > 1 or i % 2 else (400,), K, N, dtype, groups, bias=i % 4 != 3, residual=i % 5 != 1,
                          seed=i, exact=act == "relu")
    check(x, w, b, r, dy, act, torch.tensor(starts, device=DEV))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_groups_and_long_groups(dtype):
    gen = torch.Generator().manual_seed(3)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), torch.randint(0, 6000, (1023,), generator=gen).sort()[0]]).to(DEV)
    check(*make((6000,), 24, 16, dtype, 1024), "silu", starts)
    check(*make((2, 20000), 64, 32, dtype, 3), "none", torch.tensor([0, 15000, 19990], device=DEV))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
def test_few_rows_in_groups(act, dtype):
    """A handful of tokens over many groups, most of them empty, and 64 rows in one: no rounding between the backward's products."""
    starts = torch.tensor([0, 0, 2, 2, 2, 3, 3, 12, 12, 13], device=DEV)
    for shape, (K, N) in (((17,), (40, 72)), ((3, 20), (33, 50)), ((2, 17), (256, 520))):
        x, w, b, r, dy = make(shape, K, N, dtype, 9 if len(shape) == 1 else 10, seed=K)
        check(x, w, b, r, dy, act, starts)
        want = reference(x, w, b, r, dy, act, group_of_rows(starts.tolist(), w.shape[0], shape[-1]).repeat(shape[0] if len(shape) > 1 else 1).to(DEV))
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        grads = torch.autograd.grad(grouped_linear(leaves[0], leaves[1], starts, leaves[2], r, act), leaves, dy)
        for name, g in zip(("x", "weight", "bias"), grads):
            value = want[name][0].reshape(g.shape)
            # one rounding, and the fp32 arithmetic: sums of up to 520 products, values of the activations
            assert ((g.double() - value).abs() <= rounding(value, dtype) * 1.01 + 2e-5 * value.abs().max()).all(), name


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,K,N", [(65, 40, 72), (500, 33, 50), (3000, 64, 24), (19003, 136, 264), (40000, 64, 136)])
def test_bias_gradient_is_rounded_once(M, K, N, dtype):
    """The sums over rows come from the unrounded gradient of the pre-activation: one rounding, and fp32's share of a sum of M terms
    (in pieces, so far below M steps; 32 + 64 of them bound it here)."""
    x, w, b, _, dy = make((M,), K, N, dtype, residual=False, seed=M)
    leaf = b.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(fused_linear(x, w, leaf, activation="silu"), leaf, dy)
    pre = x.double() @ w.double().t() + b.double()
    terms = dy.double() * act64(pre, "silu")[1]
    value = terms.sum(0)
    slack = terms.abs().sum(0) * 2.0 ** -23 * 96 + dy.double().abs().sum(0) * 2.0 ** -20 * 4
    assert ((g.double() - value).abs() <= rounding(value, dtype) * 1.01 + slack).all()
    starts = torch.tensor([0, M // 3, M // 3 + 40, M - 7], device=DEV)
    lin = [t.unsqueeze(0).repeat(3, *(1,) * t.dim()).contiguous() for t in (w, b)]
    leaf = lin[1].requires_grad_(True)
    (g,) = torch.autograd.grad(grouped_linear(x, lin[0], starts, leaf, activation="silu"), leaf, dy)
    for e in range(3):
        rows = slice(int(starts[e]), int(starts[e + 1]))
        value = terms[rows].sum(0)
        slack = terms[rows].abs().sum(0) * 2.0 ** -23 * 96 + dy[rows].double().abs().sum(0) * 2.0 ** -20 * 4
        assert ((g[e].double() - value).abs() <= rounding(value, dtype) * 1.01 + slack).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ACTS)
def test_enough_tiles_for_every_sm(act, dtype):
    """Tall inputs, where blocks work in pairs on 256 rows: the last rows incomplete, contractions that stay in shared memory and that
    do not, widths that end inside a tile."""
    for (M, K, N), residual in (((19003, 200, 264), True), ((9607, 328, 520), False), ((19203, 256, 256), act == "none")):
        check(*make((M,), K, N, dtype, residual=residual, seed=M, exact=act == "relu"), act)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_tall_groups(act, dtype):
    """The same with groups that end inside the pairs' tiles, rows of no group before, between batch elements and behind."""
    starts = torch.tensor([100, 5003, 5003, 9000, 9391], device=DEV)
    check(*make((2, 10240), 136, 200, dtype, 4, seed=3), act, starts)
    check(*make((2, 10240), 264, 136, dtype, 5, seed=4, residual=False), act, starts)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("K,N,residual", [(64, 72, False), (64, 136, True), (200, 33, True), (72, 1200, False)])
def test_groups_of_many_tiles(K, N, residual, dtype):
    """Few groups with so many tiles each that blocks keep a group's weight: it changes inside a block's tiles, and with the batch
    element back again; aligned and odd widths, several column tiles."""
    starts = torch.tensor([300, 20011, 20100, 59000], device=DEV)
    check(*make((2, 60000), K, N, dtype, 3, seed=7, residual=residual), "silu" if residual else "none", starts)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_wide_outputs(dtype):
    """More column tiles than a block's weight could stay for."""
    check(*make((700,), 40, 6000, dtype, seed=8), "none")
    check(*make((2500,), 136, 5128, dtype, seed=9), "silu")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_weight_gradients_over_many_rows(dtype):
    """Rows enough that pairs of blocks share the weight's gradient: one group, ragged ones, and NaN in the rows behind each group's end."""
    check(*make((40003,), 264, 520, dtype, seed=5), "none")
    starts = torch.tensor([70, 15000, 15001, 15001, 20300], device=DEV)   # five entries: the last group ends before the rows do
    x, w, b, r, dy = make((2, 20480), 264, 264, dtype, 4, seed=6)
    _, grads = check(x, w, b, r, dy, "none", starts)
    for lo, hi in ((0, 70), (20300, 20480)):
        x[:, lo:hi], dy[:, lo:hi] = float("nan"), float("inf")
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    gx, gw, gb = torch.autograd.grad(grouped_linear(leaves[0], leaves[1], starts, leaves[2]), leaves, dy)
    assert torch.equal(gw, grads["weight"]) and torch.equal(gb, grads["bias"])
    assert torch.equal(gx[:, 70:20300], grads["x"][:, 70:20300]) and not gx[:, :70].any() and not gx[:, 20300:].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_other_groups_and_of_none_stay_out(dtype):
    """NaN and infinities in rows of no group, in another group's rows and weights: nothing of them reaches the group's results."""
    starts = torch.tensor([10, 75, 75, 200], device=DEV)
    x, w, b, r, dy = make((300,), 72, 40, dtype, 3, seed=4)
    clean = grouped_linear(x, w, starts, b, r, "silu")
    bad = [t.clone() for t in (x, w, b, dy)]
    for t, rows in ((bad[0], (slice(0, 10), slice(75, 300))), (bad[3], (slice(0, 10), slice(75, 300))), (bad[1], (slice(1, 3),)),
                    (bad[2], (slice(1, 3),))):
        for s in rows:
            t[s] = float("nan")
            t[s].view(-1)[::3] = float("inf")
    leaves = [t.requires_grad_(True) for t in bad[:3]]
    y = grouped_linear(*leaves[:2], starts, leaves[2], r, "silu")
    gx, gw, gb = torch.autograd.grad(y, leaves, bad[3])
    assert torch.equal(y[10:75], clean[10:75]) and torch.equal(y[:10], r[:10]) and torch.equal(y[200:], r[200:])
    assert y[75:200].isnan().any()
    ref = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(grouped_linear(*ref[:2], starts, ref[2], r, "silu"), ref, dy)
    assert torch.equal(gx[10:75], want[0][10:75]) and not gx[:10].any() and not gx[200:].any()
    assert torch.equal(gw[0], want[1][0]) and torch.equal(gb[0], want[2][0])
    assert not gw[1].any() and not gb[1].any()      # no rows: zero, whatever its weight


@pytest.mark.parametrize("dtype", DTYPES)
def test_special_values_pass_through(dtype):
    x, w, b, r, dy = make((130,), 64, 32, dtype, seed=5)
    x[3, 7], x[64] = float("nan"), float("inf")
    y = fused_linear(x, w, b, activation="relu")
    assert y[3].isnan().all() and torch.isfinite(y[65:]).all()
    want = x.double() @ w.double().t() + b.double()
    assert torch.equal(y[64].isnan(), want[64].isnan())
    keep = ~want[64].isnan()
    assert torch.equal(y[64][keep].double(), want[64][keep].clamp_min(0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
    """Transposed and sliced operands, a broadcast gradient, storage that starts off any vector's boundary."""
    x, w, b, r, dy = make((96,), 64, 48, dtype, seed=6)
    y, grads = check(x, w, b, r, dy, "silu")
    wide = torch.zeros(96, 131, device=DEV, dtype=dtype)
    wide[:, 3:67] = x
    wt = w.t().contiguous().t()

    def shifted(t):
        s = torch.zeros(t.numel() + 1, device=DEV, dtype=dtype)[1:].view(t.shape)
        return s.copy_(t)

    for ops in ((wide[:, 3:67], wt, b.expand(48), r.t().contiguous().t()), tuple(map(shifted, (x, w, b, r)))):
        leaves = [t.detach().requires_grad_(True) for t in ops]
        y2 = fused_linear(*leaves, "silu")
        g2 = torch.autograd.grad(y2, leaves, shifted(dy))
        compare(y2, reference(x, w[None], b[None], r, dy, "silu")["y"], "y")
        want = reference(x, w[None], b[None], r, dy, "silu")
        for n, g in zip(("x", "weight", "bias"), g2):
            compare(g, want[n], n)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    ones = torch.autograd.grad(fused_linear(*leaves, activation="silu").sum(), leaves)
    want = reference(x, w[None], b[None], None, torch.ones_like(dy), "silu")
    for n, g in zip(("x", "weight", "bias"), ones):
        compare(g, want[n], n)


def test_no_rows():
    for dtype in DTYPES:
        x, w, b, r, dy = make((0,), 16, 24, dtype)
        leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
        y = fused_linear(*leaves, "gelu")
        assert y.shape == (0, 24)
        gx, gw, gb, gr = torch.autograd.grad(y, leaves, dy)
        assert gx.shape == (0, 16) and gr.shape == (0, 24) and not gw.any() and not gb.any()


def test_only_wanted_gradients():
    x, w, b, r, dy = make((200,), 64, 72, torch.bfloat16, seed=7)
    want = check(x, w, b, r, dy, "gelu")[1]
    for names in (("x",), ("weight",), ("bias",), ("residual",), ("weight", "residual")):
        tensors = dict(x=x.clone(), weight=w.clone(), bias=b.clone(), residual=r.clone())
        for n in names:
            tensors[n].requires_grad_(True)
        y = fused_linear(*tensors.values(), "gelu")
        for n, g in zip(names, torch.autograd.grad(y, [tensors[n] for n in names], dy)):
            assert torch.equal(g, want[n]), n


def test_x_as_its_own_residual():
    x, w, b, _, dy = make((77,), 48, 48, torch.float32, seed=8)
    leaf = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(fused_linear(leaf, w, b, leaf, "silu"), leaf, dy)
    other = x.clone().requires_grad_(True)
    (gx,) = torch.autograd.grad(fused_linear(other, w, b, activation="silu"), other, dy)
    assert torch.equal(g, gx + dy)


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_gradients_against_differences(act):
    """Directional derivative of sum(c * y) from two forwards in fp32.  Bound: twice the forward's bound over 2h, plus h^2/6 of the
    third derivative (below 3 for these functions) along the direction."""
    x, w, b, _, c = make((50,), 30, 20, torch.float32, seed=9)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(fused_linear(*leaves, activation=act), leaves, c)
    h = 2.0 ** -6
    gen = torch.Generator(device=DEV).manual_seed(10)
    for i, leaf in enumerate(leaves):
        d = torch.randn(leaf.shape, generator=gen, device=DEV) * 0.5
        moved = [[t.detach() + s * h * d if j == i else t.detach() for j, t in enumerate(leaves)] for s in (1, -1)]
        ys = [fused_linear(*m, activation=act).double() for m in moved]
        difference = ((ys[0] - ys[1]) * c.double()).sum().item() / (2 * h)
        # the points moved to are rounded to fp32, so take the step that was made
        made = (moved[0][i].double() - moved[1][i].double()) / (2 * h)
        along = (grads[i].double() * made).sum().item()
        ref = reference(moved[0][0], moved[0][1][None], moved[0][2][None], None, c, act)
        here = reference(leaves[0], leaves[1][None], leaves[2][None], None, c, act)
        dpre = {0: lambda: made @ leaves[1].detach().double().t(), 1: lambda: leaves[0].detach().double() @ made.t(),
                2: lambda: made.expand(50, 20)}[i]()
        name = ("x", "weight", "bias")[i]
        bound = (2 * (ref["y"][1] * c.double().abs()).sum().item() / (2 * h) * 1.1 + h * h / 6 * 3 * (c.double().abs() * dpre.abs() ** 3).sum().item()
                 + (here[name][1].reshape(made.shape) * made.abs()).sum().item())
        assert abs(difference - along) <= bound
        assert bound <= 0.2 * max(abs(along), (grads[i].double().norm() * made.norm()).item())   # the bound says something


def test_repeats_are_equal_and_streams_are_kept():
    x, w, b, r, dy = make((3000,), 136, 264, torch.bfloat16, seed=11)
    _, first = check(x, w, b, r, dy, "gelu")
    side = torch.cuda.Stream()
    for _ in range(3):
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(2_000_000)
            late = x * 1                      # made on the side stream behind a delay
            leaves = [t.detach().requires_grad_(True) for t in (late, w, b)]
            y = fused_linear(*leaves, r, "gelu")
            grads = torch.autograd.grad(y, leaves, dy)
        side.synchronize()
        for n, g in zip(("x", "weight", "bias"), grads):
            assert torch.equal(g, first[n]), n


def test_calls_from_a_thread_that_has_not_used_the_device():
    import threading

    x, w, b, r, dy = make((200,), 64, 72, torch.bfloat16, seed=16)
    want, grads = check(x, w, b, r, dy, "none")
    got = []

    def call():
        from ops3d_b200 import _C

        try:
            got.append(_C.linear_forward(x, w, b, r, None, 0))
            got.extend(_C.linear_backward(x, w, b, None, dy, 0, True, True, True))
        except RuntimeError as e:
            got.append(e)

    thread = threading.Thread(target=call)
    thread.start()
    thread.join()
    assert len(got) == 4 and not isinstance(got[-1], RuntimeError), got[-1]
    for a, e in zip(got, (want, grads["x"], grads["weight"], grads["bias"])):
        assert torch.equal(a, e)


def test_captured_training_pass_follows_its_inputs():
    """One graph of forward and backward; inputs and group boundaries change between replays.  No eager graph of the same leaves may
    live meanwhile: torch ties a leaf's accumulation node to the stream of its first use, and a capture that meets the default
    stream's is invalid, whatever the operator."""
    x, w, b, r, dy = make((2, 500), 64, 72, torch.float16, 3, seed=12)
    starts = torch.tensor([0, 100, 400], device=DEV)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def step():
        y = grouped_linear(leaves[0], leaves[1], starts, leaves[2], r, "silu")
        return (y, *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.cuda.graph(second):
        out2 = step()
    for boundaries, seed in (([0, 100, 400], 20), ([30, 31, 31], 21), ([0, 0, 0], 22)):
        with torch.no_grad():
            starts.copy_(torch.tensor(boundaries))
            x.copy_(make((2, 500), 64, 72, torch.float16, 3, seed=seed)[0])
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        eager = step()
        for a, a2, e in zip(out, out2, eager):
            assert torch.equal(a, e) and torch.equal(a2, e)


@pytest.mark.parametrize("M", [3, 200, 20000])
def test_neighbours_in_the_stream(M):
    """Copies, fills and kernels right before and after, eager and captured: the operators' kernels are set up early but see what came
    before, and what comes after sees theirs."""
    x, w, b, r, dy = make((M,), 64, 136, torch.bfloat16, seed=17)
    inputs = [make((M,), 64, 136, torch.bfloat16, seed=s)[0] for s in (18, 19, 20)]
    want = [fused_linear(v, w, b, r, "silu") for v in inputs]
    torch.cuda.synchronize()
    buffer, out, mark = torch.empty_like(x), torch.empty_like(r), torch.empty(1 << 20, device=DEV)

    def step(v):
        mark.zero_()
        buffer.copy_(v)                                   # a copy, not a kernel
        y = fused_linear(buffer, w, b, r, "silu")
        buffer.zero_()                                    # while the product may still be running
        out.copy_(y)
        y.fill_(float("nan"))
        return out

    for _ in range(20):
        for v, e in zip(inputs, want):
            assert torch.equal(step(v), e)
    source = inputs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(source)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(source)
    for _ in range(5):
        for v, e in zip(inputs, want):
            source.copy_(v)
            graph.replay()
            assert torch.equal(out, e)


def test_under_autocast_and_checkpointing():
    """fp32 parameters beside the 16-bit tensors that autocast makes, and the operators inside a recomputed segment."""
    from torch.utils.checkpoint import checkpoint

    torch.manual_seed(3)
    ff = FeedForward(32, 64, "gelu").to(DEV)
    x = torch.randn(100, 32, device=DEV)
    with torch.autocast("cuda", torch.bfloat16):
        h = torch.nn.functional.linear(x, torch.eye(32, device=DEV))
        y = ff(h)
    assert h.dtype == torch.bfloat16 and y.dtype == torch.bfloat16
    leaf = x.clone().requires_grad_(True)
    plain = torch.autograd.grad(ff(leaf).square().sum(), [leaf, *ff.parameters()])
    again = torch.autograd.grad(checkpoint(ff, leaf, use_reentrant=False).square().sum(), [leaf, *ff.parameters()])
    for a, e in zip(again, plain):
        assert torch.equal(a, e)


def test_graphs_and_threads_at_once():
    """Captured passes replayed on two streams at once, and threads on streams of their own and on a shared one, give what a pass
    alone gives: no workspace is shared."""
    starts = torch.tensor([0, 100, 100, 900, 2000, 9000], device="cuda")
    inputs = []
    for k in range(2):
        torch.manual_seed(k)
        x = torch.randn(9500, 72, device="cuda", dtype=torch.bfloat16).requires_grad_()
        inputs.append((x, torch.randn(6, 136, 72, device="cuda", dtype=torch.bfloat16).requires_grad_()))

    def grads(k):
        x, w = inputs[k]
        return torch.autograd.grad(grouped_linear(x, w, starts, None, None, "gelu").square().sum(), (x, w))

    wants = [grads(k) for k in range(2)]
    torch.cuda.synchronize()
    differing = []

    def repeat(stream, k):
        with torch.cuda.stream(stream):
            for _ in range(20):
                if not all(torch.equal(a, b) for a, b in zip(grads(k), wants[k])):
                    differing.append(k)

    threads = [threading.Thread(target=repeat, args=(torch.cuda.Stream() if i % 2 else torch.cuda.default_stream(), i // 2)) for i in range(4)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not differing

    captured = []
    for k in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = grads(k)
        captured.append((graph, results, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, _, stream in captured:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for (_, results, _), want in zip(captured, wants):
        assert all(torch.equal(a, b) for a, b in zip(results, want))


def test_refusals():
    x, w, b, r, dy = make((10,), 16, 24, torch.bfloat16)
    starts = torch.tensor([0], device=DEV)
    cases = [
        (lambda: fused_linear(x, w.float()), "dtype of x"), (lambda: fused_linear(x, w, b.float()), "dtype of x"),
        (lambda: fused_linear(x, w, b, r.float()), "dtype of x"), (lambda: fused_linear(x.double(), w.double()), "float32, float16 or bfloat16"),
        (lambda: fused_linear(x, w.cpu()), "CUDA tensor"), (lambda: fused_linear(x[:, :8], w), "features like weight"),
        (lambda: fused_linear(x, w[None]), "out_features, in_features"), (lambda: fused_linear(x, w, b[:5]), "bias must be"),
        (lambda: fused_linear(x, w, b, r[:5]), "shape of the output"), (lambda: fused_linear(x, w, b, r[:1]), "shape of the output"),
        (lambda: fused_linear(x, w[:0]), "must not be empty"), (lambda: fused_linear(x[:, :0], w[:, :0]), "must not be empty"),
        (lambda: grouped_linear(x, w, starts), "groups, out_features, in_features"),
        (lambda: grouped_linear(x, w[None], starts.int()), "int64"), (lambda: grouped_linear(x, w[None], starts[None]), "one-dimensional"),
        (lambda: grouped_linear(x, w[None], starts.cpu()), "same device"),
        (lambda: grouped_linear(x, w[None].expand(3, 24, 16), starts), "one entry per group"),
        (lambda: grouped_linear(x[None, None], w[None], starts), "rows, in_features"),
        (lambda: grouped_linear(x, w[None], starts, b), "bias must be"),
        (lambda: grouped_linear(x, w[None].expand(1025, 24, 16), starts.expand(1025)), "compiled-in capacity"),
    ]
    for call, match in cases:
        with pytest.raises(RuntimeError, match=match):
            call()
    leaf = x.clone().requires_grad_(True)
    y = fused_linear(leaf, w, b, activation="silu")
    (g,) = torch.autograd.grad(y, leaf, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
    y = fused_linear(leaf, w, b)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()


def test_saved_tensors_are_version_checked():
    x, w, b, _, dy = make((10,), 16, 24, torch.float32)
    leaf = x.clone().requires_grad_(True)
    y = fused_linear(leaf, w, b)
    w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_offsets_beyond_32_bits(dtype):
    """More than 2^31 elements of x (and of y): the last rows are where a 32-bit offset would go wrong."""
    K, N = 1032, 1024
    M = 2 ** 31 // N + 300
    gen = torch.Generator(device=DEV).manual_seed(13)
    x = torch.zeros(M, K, dtype=dtype, device=DEV)
    x[-300:] = torch.randn(300, K, generator=gen, device=DEV).to(dtype)
    w = (torch.randn(N, K, generator=gen, device=DEV) / 32).to(dtype)
    dy = torch.zeros(M, N, dtype=dtype, device=DEV)
    dy[-300:] = torch.randn(300, N, generator=gen, device=DEV).to(dtype)
    leaves = [t.requires_grad_(True) for t in (x, w)]
    y = fused_linear(*leaves, activation="silu")
    gx, gw = torch.autograd.grad(y, leaves, dy)
    want = reference(x[-300:], w[None], None, None, dy[-300:], "silu")
    compare(y[-300:], want["y"], "y")
    compare(gx[-300:], want["x"], "grad_x")
    value, bound = want["weight"]
    # the zero rows add nothing, but the sum has M terms
    compare(gw, (value, bound * (1 + 300 / 300)), "grad_weight")
    assert not y[:1000].any() and not gx[:1000].any()


def test_feed_forward_and_layer_together():
    """The layer with its own level projections and residual, then a feed-forward per level: outputs and all gradients against the
    same in 64-bit products around the operator."""
    from oracle.fda_oracle import level_start_index_of, ms_deform_attn_core_pytorch_3d
    from ops3d_b200.msda3d import MSDeformAttn3D

    torch.manual_seed(0)
    shapes = torch.tensor([(6, 8, 10), (3, 4, 5)])
    lsi = level_start_index_of(shapes)
    N, B, C, G, L, K = int(shapes.prod(1).sum()), 2, 64, 4, 2, 4
    layer = MSDeformAttn3D(C, L, G, K, level_value_proj=True).to(DEV)
    ffn = FeedForward(C, 96, "gelu", n_groups=L).to(DEV)
    with torch.no_grad():
        layer.sampling_offsets.weight.normal_(0, 0.05)
        layer.attention_weights.weight.normal_(0, 0.3)
        for p in (layer.value_proj.bias, layer.output_proj.bias, ffn.bias1, ffn.bias2):
            p.normal_(0, 0.1)
    src = torch.randn(B, N, C, device=DEV, requires_grad=True)
    ref = torch.rand(B, N, L, 3, device=DEV)
    params = [*layer.parameters(), *ffn.parameters()]
    out = ffn(layer(src, ref, src, shapes.to(DEV), lsi.to(DEV), residual=src), lsi.to(DEV))
    dy = torch.randn_like(out)
    got = [out, *torch.autograd.grad(out, [src, *params], dy)]

    p64 = {n: p.detach().double().cpu().requires_grad_(True) for n, p in
           [*((f"a.{n}", p) for n, p in layer.named_parameters()), *((f"f.{n}", p) for n, p in ffn.named_parameters())]}
    s64 = src.detach().double().cpu().requires_grad_(True)
    owner = group_of_rows(lsi.tolist(), L, N)

    def per_level(x, w, b):
        return torch.stack([x[:, n] @ w[owner[n]].t() + b[owner[n]] for n in range(N)], 1)

    value = per_level(s64, p64["a.value_proj.weight"], p64["a.value_proj.bias"]).view(B, N, G, -1)
    off = (s64 @ p64["a.sampling_offsets.weight"].t() + p64["a.sampling_offsets.bias"]).view(B, N, G, L, K, 3)
    logits = (s64 @ p64["a.attention_weights.weight"].t() + p64["a.attention_weights.bias"]).view(B, N, G, L * K)
    loc = ref.double().cpu()[:, :, None, :, None, :] + off / shapes.flip(-1).double()[None, None, None, :, None, :]
    attended = ms_deform_attn_core_pytorch_3d(value, shapes, loc, logits.softmax(-1).view(B, N, G, L, K))
    mid = s64 + attended @ p64["a.output_proj.weight"].t() + p64["a.output_proj.bias"]
    hidden = torch.nn.functional.gelu(per_level(mid, p64["f.weight1"], p64["f.bias1"]))
    want_out = mid + per_level(hidden, p64["f.weight2"], p64["f.bias2"])
    want = [want_out, *torch.autograd.grad(want_out, [s64, *p64.values()], dy.double().cpu())]
    # fp32 throughout: the layer's own bound of 2e-4 of the largest value (test_gpu_msda3d.py)
    for g, v in zip(got, want):
        assert g.shape == v.shape
        assert (g.double().cpu() - v).abs().max().item() <= 2e-4 * max(1.0, v.abs().max().item())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_modules_in_16_bits(dtype):
    """fp32 parameters beside 16-bit inputs are taken in the inputs' type."""
    x = torch.randn(2, 50, 32, device=DEV).to(dtype)
    lsi = torch.tensor([0, 40], device=DEV)
    lin = GroupedLinear(2, 32, 24).to(DEV)
    assert torch.equal(lin(x, lsi), grouped_linear(x, lin.weight.to(dtype), lsi, lin.bias.to(dtype)))
    ff = FeedForward(32, 64, "silu").to(DEV)
    y = ff(x)
    assert y.dtype == dtype and y.shape == x.shape
    y.float().square().sum().backward()
    assert all(p.grad is not None and p.grad.dtype == torch.float32 and torch.isfinite(p.grad).all() for p in ff.parameters())
