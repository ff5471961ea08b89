"""The gradients of layer norm's parameters: sums over many rows that miss none.

A row passes through few additions on its way into a sum, u = 2^-24 each: those of a team's rows (a block has eight teams or more up to 256
features, and there are 296 blocks or more where rows are that many; wider rows have 144 blocks or more, beyond 8192 features 64 parts), up to 64 teams
of a block, 3 steps over a warp, and 10 over the blocks.  What one lost row, team or block takes away is far more.
"""
import pytest
import torch

from ops3d_b200 import layer_norm
from test_gpu_layer_norm import BF16, DEV, F16, F32, MORE, U, make, reference

pytestmark = pytest.mark.gpu

CASES = [(40000, 64, BF16, BF16), (40001, 8, F16, None), (30011, 5, BF16, None), (25003, 1, F32, None), (20001, 259, BF16, None), (9001, 250, F16, F32),
         (5003, 131, F32, F32), (12000, 256, BF16, F32), (7001, 512, BF16, BF16), (3001, 640, F16, None), (3000, 1024, BF16, BF16), (1501, 4099, BF16, None),
         (701, 8192, F32, None), (700, 8191, F16, F32), (301, 9001, BF16, F32)]


def chain(rows, width):
    teams = 8 * 296 if width <= 256 else 144 if width <= 8192 else 64
    return -(-rows // teams) + 1 + 64 + 3 + 10


def parameter_gradients(x, w, b, r, dy):
    leaves = [t.detach().requires_grad_(True) for t in (w, b)]
    return torch.autograd.grad(layer_norm(x, *leaves, residual=r), leaves, dy)


def z_of(x, r, eps=1e-5):
    s = x.double() if r is None else x.double() + r.double()
    d = s - s.mean(-1, keepdim=True)
    return d / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)


@pytest.mark.parametrize("rows,width,dtype,residual", CASES, ids=str)
def test_sums_are_off_by_a_few_additions(rows, width, dtype, residual):
    x, w, b, r, dy, _ = make((rows, width), dtype, F32, residual, seed=rows)
    dw, db = parameter_gradients(x, w, b, r, dy)
    want = reference(x, w, b, r, 1e-5, dy)
    magnitude = (dy.double() * z_of(x, r)).abs().sum(0)
    value, bound = want["weight"]
    bound = bound - (rows + 2) * U * magnitude + chain(rows, width) * U * magnitude        # z's own errors, and the additions
    worst = ((dw.double() - value).abs() / (bound * MORE + U * value.abs()).clamp_min(1e-300)).max().item()
    assert worst <= 1.0, f"weight: {worst:.3f} of the bound"
    value, magnitude = want["bias"][0], dy.double().abs().sum(0)
    worst = ((db.double() - value).abs() / (chain(rows, width) * U * magnitude * MORE + U * value.abs())).max().item()
    assert worst <= 1.0, f"bias: {worst:.3f} of the bound"


@pytest.mark.parametrize("rows,width,dtype,residual", CASES, ids=str)
def test_sums_of_whole_numbers_are_exact(rows, width, dtype, residual):
    """Sums below 2^24 have no rounding, in whatever order: every row is in them, once."""
    x, w, b, r, _, _ = make((rows, width), dtype, F32, residual, seed=1)
    dy = torch.randint(-3, 4, (rows, width), device=DEV, generator=torch.Generator(device=DEV).manual_seed(rows)).to(dtype)
    _, db = parameter_gradients(x, w, b, r, dy)
    assert torch.equal(db.double(), dy.double().sum(0))
    if width in (8, 64, 256, 512, 1024):
        # rows of +-a, a power of two: z is +-1 to the last bit where eps is 0 and the width divides exactly
        sign = (torch.arange(width, device=DEV) % 2 * 2 - 1) * torch.where(torch.arange(rows, device=DEV) % 3 == 0, -1, 1)[:, None]
        x = (sign * 2.0 ** (torch.arange(rows, device=DEV) % 5 - 2)[:, None]).to(dtype)
        weight = w.detach().requires_grad_(True)
        (dw,) = torch.autograd.grad(layer_norm(x, weight, b, eps=0.0), weight, dy)
        assert torch.equal(dw.double(), (dy.double() * sign).sum(0))


@pytest.mark.parametrize("rows,width,dtype,residual", CASES, ids=str)
def test_each_row_reaches_the_sums(rows, width, dtype, residual):
    """A gradient in one row alone: its product is the whole sum.  Rows of the first and the last blocks, teams and stages, and some between."""
    x, w, b, r, dy, _ = make((rows, width), dtype, F32, residual, seed=2)
    gen = torch.Generator().manual_seed(rows)
    picked = sorted({0, 1, 7, 8, 295, 296, 443, 444, *range(rows - 9, rows), *torch.randint(0, rows, (12,), generator=gen).tolist()})
    for row in (r_ for r_ in picked if r_ < rows):
        only = torch.zeros_like(dy)
        only[row] = dy[row]
        dw, db = parameter_gradients(x, w, b, r, only)
        assert torch.equal(db, dy[row].float())
        one = slice(row, row + 1)
        value, bound = reference(x[one], w, b, None if r is None else r[one], 1e-5, dy[one])["weight"]
        assert ((dw.double() - value).abs() <= bound * MORE + U * value.abs()).all(), row
