"""Linear operators over small whole numbers, whose products and sums are exact in fp32 in any order as long as they stay below
2^24: every result has to be the whole number, rounded once to the tensors' type.  A row, a block or a sum of a piece that is left out,
taken twice or taken from another group shows in every element that it belongs to, however long the sum.

Values are -2 .. 2, so a sum of n products is at most 4 n: 2^24 is reached from 4 million terms on.
"""
import pytest
import torch

from ops3d_b200 import capi, fused_linear, grouped_linear

pytestmark = pytest.mark.gpu

DEV = "cuda"
NARROW = [torch.float16, torch.bfloat16]
DTYPES = [torch.float32, *NARROW]


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    torch.cuda.synchronize()
    assert capi.load().fda_linear_timeouts() == 0


def whole(gen, *shape):
    return torch.randint(-2, 3, shape, generator=gen, device=DEV).double()


def operands(lead, K, N, groups=None, seed=0):
    """x, weight, bias, residual and the output's gradient, in 64 bits."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    g = () if groups is None else (groups,)
    return whole(gen, *lead, K), whole(gen, *g, N, K), whole(gen, *g, N), whole(gen, *lead, N), whole(gen, *lead, N)


def expected(x, w, b, r, dy, starts=None, relu=False):
    """y, grad_x, grad_weight, grad_bias in 64 bits; starts: ascending, one entry more than groups."""
    K, N = x.shape[-1], w.shape[-2]
    rows = x.shape[-2]
    batch = x.numel() // (rows * K)
    spans = [(0, rows)] if starts is None else list(zip(starts[:-1], starts[1:]))
    x, dy = x.reshape(batch, rows, K), dy.reshape(batch, rows, N)
    y = torch.zeros_like(dy) if r is None else r.reshape(batch, rows, N).clone()
    gx, gw, gb = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    for e, (lo, hi) in enumerate(spans):
        we, be = (w, b) if starts is None else (w[e], b[e])
        xe, ge = x[:, lo:hi].reshape(-1, K), dy[:, lo:hi].reshape(-1, N)
        pre = xe @ we.t() + be
        if relu:
            ge = ge * (pre > 0)
            pre = pre.clamp_min(0)
        y[:, lo:hi] += pre.view(batch, hi - lo, N)
        gx[:, lo:hi] = (ge @ we).view(batch, hi - lo, K)
        (gw if starts is None else gw[e]).copy_(ge.t() @ xe)
        (gb if starts is None else gb[e]).copy_(ge.sum(0))
    return y, gx, gw, gb


def run(x, w, b, r, dy, dtype, starts=None, relu=False):
    leaves = [t.to(dtype).requires_grad_(True) for t in (x, w, b)]
    r = None if r is None else r.to(dtype)
    act = "relu" if relu else "none"
    if starts is None:
        y = fused_linear(*leaves, r, act)
    else:
        y = grouped_linear(leaves[0], leaves[1], torch.tensor(starts, device=DEV), leaves[2], r, act)
    return (y, *torch.autograd.grad(y, leaves, dy.to(dtype)))


def same(got, want, dtype):
    for name, g, v in zip(("y", "grad_x", "grad_weight", "grad_bias"), got, want):
        assert v.abs().max().item() < 2 ** 24
        bad = (g != v.to(dtype).view(g.shape)).sum().item()
        assert bad == 0, f"{name}: {bad} of {g.numel()} elements"


# Weight gradients of which pairs of blocks take 64 rows at a time, and both have to clear the rows behind a group's end: groups that
# end anywhere inside a block, with every batch element; in pieces whose sums are added, and whole.
PAIRED = {
    "pieces": ((2, 20480), 264, 264, [70, 15000, 15001, 15001, 20301]),
    "whole": ((2, 1500), 2048, 1800, [3, 600, 601, 999, 1400]),
    "three elements": ((3, 9001), 520, 264, [0, 4001, 4102, 9000]),
}


@pytest.mark.parametrize("dtype", NARROW)
@pytest.mark.parametrize("kind", PAIRED)
def test_rows_behind_a_group_stay_out_of_both_blocks(kind, dtype):
    lead, K, N, starts = PAIRED[kind]
    x, w, b, r, dy = operands(lead, K, N, len(starts) - 1, seed=1)
    want = expected(x, w, b, None, dy, starts)
    for t in (x, dy):   # rows of no group
        t[..., :starts[0], :], t[..., starts[-1]:, :] = float("nan"), float("inf")
    for _ in range(5):
        same(run(x, w, b, None, dy, dtype, starts), want, dtype)


@pytest.mark.parametrize("dtype", NARROW)
@pytest.mark.parametrize("grouped", [False, True], ids=["one", "groups"])
def test_extra_rows_of_one_tile_never_reach_another(grouped, dtype):
    """A residual, and in the backward the output's gradient, pass through a buffer that is filled again while the tile before is still
    being written: tall inputs, several tiles a pair of blocks, short contractions (the buffer's turn comes soonest)."""
    starts = [130, 9001, 9001, 30011] if grouped else None
    lead = (2, 30011) if grouped else (60011,)
    for K, N in ((16, 520), (200, 264)):
        ops = operands(lead, K, N, 3 if grouped else None, seed=K)
        want = expected(*ops, starts, relu=True)
        for _ in range(5):
            same(run(*ops, dtype, starts, relu=True), want, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_groups_that_just_need_several_pieces(dtype):
    """As many groups as the rows allow that are one row longer than a piece, the rest hardly any: all partial sums that a call can have.
    (16-bit: pieces of 512 rows; fp32: 256 rows an element of the batch are a block, and with 9 elements each row is a piece.)"""
    sizes = [513, 0, 513, 1, 513, 2, *[1] * 40, 0, 513, 3, 513, *[0] * 100]
    starts = [5]
    for n in sizes:
        starts.append(starts[-1] + n)
    ops = operands((starts[-1] + 20,), 264, 520, len(sizes), seed=2)
    same(run(*ops[:3], None, ops[4], dtype, starts), expected(*ops[:3], None, ops[4], starts), dtype)
    sizes = [1, 3, 0, 1, 2, 0, 0, 1]
    starts = [1]
    for n in sizes:
        starts.append(starts[-1] + n)
    ops = operands((40, starts[-1] + 1), 72, 136, len(sizes), seed=3)
    same(run(*ops[:3], None, ops[4], dtype, starts), expected(*ops[:3], None, ops[4], starts), dtype)


# lead, inputs, outputs, groups' start indices, relu.  Chosen so that every form of the products over many rows is met: weights that stay in
# shared memory and that stream, one block and pairs, pieces and whole groups, odd widths, few rows.
TALL = [
    ((40003,), 264, 520, None, False), ((40003,), 264, 1032, None, True), ((70001,), 64, 72, None, True), ((30011,), 131, 99, None, True),
    ((2, 60000), 64, 72, [300, 20011, 20100, 59000], False), ((2, 60000), 136, 72, [300, 20011, 20100, 59000], True),
    ((3, 15013), 264, 264, [0, 7001, 7001, 7002, 15013], True), ((2, 30011), 33, 50, [11, 20000, 30011], True),
    ((2, 4099), 1032, 1800, [0, 1000, 2500, 4001], False), ((9001,), 2056, 1032, None, True), ((61,), 264, 520, None, True),
    ((700, 50), 72, 1032, [3, 20, 21, 47], True), ((3000, 9), 40, 264, [0, 4, 4, 9], True), ((2, 31), 72, 136, [1, 2, 2, 25], True), ((1,), 1032, 2056, None, True),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", TALL, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}-{'groups' if c[3] else 'one'}-{'relu' if c[4] else 'none'}")
def test_every_element_over_many_rows(case, dtype):
    """All four gradients and the output, element for element: no row is lost, doubled or taken from elsewhere."""
    lead, K, N, starts, relu = case
    ops = operands(lead, K, N, None if starts is None else len(starts) - 1, seed=K + N)
    same(run(*ops, dtype, starts, relu), expected(*ops, starts, relu), dtype)


def test_as_many_rows_as_there_may_be():
    """2^31 - 1 rows of one feature: a count of them that is rounded up passes 31 bits.  Rows that matter lie at both ends."""
    M, dtype = 2 ** 31 - 1, torch.bfloat16
    x, dy = torch.zeros(M, 1, dtype=dtype, device=DEV), torch.zeros(M, 1, dtype=dtype, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(4)
    ends = [slice(0, 300), slice(M - 300, M)]
    for rows in ends:
        x[rows], dy[rows] = whole(gen, 300, 1).to(dtype), whole(gen, 300, 1).to(dtype)
    w, b = torch.full((1, 1), 2.0, dtype=dtype, device=DEV), torch.ones(1, dtype=dtype, device=DEV)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = fused_linear(*leaves, activation="relu")
    gx, gw, gb = torch.autograd.grad(y, leaves, dy)
    assert (y[300:M - 300] == 1).all() and not gx[300:M - 300].any()
    xe, ge = (torch.cat([t.detach()[rows].double() for rows in ends]) for t in (x, dy))
    pre = 2 * xe + 1
    ge = ge * (pre > 0)
    assert torch.equal(torch.cat([y[rows] for rows in ends]).double(), pre.clamp_min(0))
    assert torch.equal(torch.cat([gx[rows] for rows in ends]).double(), 2 * ge)
    assert gw.item() == (ge * xe).sum().to(dtype).item() and gb.item() == ge.sum().to(dtype).item()
