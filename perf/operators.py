"""Performance cases of the linear operators: a matrix product with bias, activation and residual in its epilogue, for one
weight (``fused_linear``) and for one weight per ragged group of rows (``grouped_linear``), forward and training.

    pre = x @ weight^T + bias,   y = act(pre) + residual
    g = dy * act'(pre),   dx = g @ weight,   dweight = g^T @ x,   dbias = sum of g's rows,   dresidual = dy

``listed()`` holds named cases, ``draw(rng)`` further ones of the same ranges; ``prepare`` builds what a program has in hand
before the call, ``run`` is one pass (``own``: through this package, else in elementary torch operations in 32 bits),
``exact`` the same from the definition in 64 bits, ``work`` the bytes and operations that a pass cannot do without.

A case is a dict of plain values.  ``rows`` is the number of rows of ``x``, or for the grouped operator the rows of each group
("4096+512", one batch element; zero is an empty group); ``batch`` elements repeat the same groups; ``tail`` rows behind the
last group belong to none.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}

# What a drawn case may cost at most, all below the largest listed one.
MAX_PRODUCTS = 2 ** 35     # rows * inputs * outputs
MAX_ELEMENTS = 2 ** 28     # of x, of y, of all weights


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # One token through the first half of a feed-forward: latency of a single call.
        dict(name="one token bf16 infer", op="linear", mode="infer", rows=1, inputs=256, outputs=1024, act="gelu",
             bias=True, residual=False, dtype="bf16"),
        # 200 object queries of four images through the same, training in half precision.
        dict(name="decoder queries f16 train", op="linear", mode="train", rows=800, inputs=256, outputs=1024, act="gelu",
             bias=True, residual=False, dtype="f16"),
        # Full precision, every size odd: a small model's head.
        dict(name="ragged f32 train", op="linear", mode="train", rows=3001, inputs=99, outputs=131, act="silu",
             bias=True, residual=True, dtype="f32"),
        # Features with three coordinates appended: rows that no 16-byte vector divides.
        dict(name="odd widths bf16 train", op="linear", mode="train", rows=9473, inputs=259, outputs=250, act="gelu_tanh",
             bias=True, residual=True, dtype="bf16"),
        # First half of an encoder's feed-forward over four pyramids of 37 376 cells.
        dict(name="feed-forward up bf16 infer", op="linear", mode="infer", rows=149504, inputs=256, outputs=1024, act="relu",
             bias=True, residual=False, dtype="bf16"),
        # The same in training, over one pyramid of 73 728 cells.
        dict(name="feed-forward up f16 train", op="linear", mode="train", rows=73728, inputs=256, outputs=1024, act="gelu",
             bias=True, residual=False, dtype="f16"),
        # Second half, with the residual connection.
        dict(name="feed-forward down bf16 train", op="linear", mode="train", rows=73728, inputs=1024, outputs=256, act="none",
             bias=True, residual=True, dtype="bf16"),
        # The attention layer's output projection with its residual, one tile of 598 016 cells.
        dict(name="output projection bf16 train", op="linear", mode="train", rows=598016, inputs=256, outputs=256, act="none",
             bias=True, residual=True, dtype="bf16"),
        # A handful of tokens sorted by expert, most experts without any.
        dict(name="expert tokens bf16 infer", op="grouped", mode="infer", rows="0+2+0+0+1+0+0+0+0+0+1+0+0+0+3+0+0+0+0+0+0+0+0+1",
             batch=1, tail=0, inputs=256, outputs=1024, act="gelu", bias=True, residual=False, dtype="bf16"),
        # Value projection with a weight of its own for each level of a small pyramid.
        dict(name="level values bf16 infer", op="grouped", mode="infer", rows="4096+512", batch=2, tail=0, inputs=256,
             outputs=256, act="none", bias=True, residual=False, dtype="bf16"),
        # Unevenly loaded experts in training, one without rows, padding behind the last.
        dict(name="experts f16 train", op="grouped", mode="train",
             rows="1211+37+4096+0+953+2048+511+640+1+1777+300+129+2500+64+801+1190", batch=1, tail=126, inputs=256,
             outputs=1024, act="silu", bias=True, residual=False, dtype="f16"),
        # Value projection per level over the pyramid of a 256x512x2048 tile, two of them, training.
        dict(name="level values bf16 train", op="grouped", mode="train", rows="524288+65536+8192", batch=2, tail=0, inputs=256,
             outputs=256, act="none", bias=True, residual=False, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng):
    """A feature width: mostly a multiple of 8, as layers have them, sometimes any number."""
    n = _log_int(rng, 16, 2048)
    return n if rng.random() < 0.25 else max(8, n // 8 * 8)


def draw(rng):
    while True:
        case = dict(op=rng.choice(["linear", "grouped"]), mode=rng.choice(["infer", "train"]))
        rows = 1 if rng.random() < 0.1 else _log_int(rng, 1, 300000)
        batch = 1
        if case["op"] == "linear":
            case["rows"] = rows
        else:
            groups = _log_int(rng, 1, 64)
            batch = rng.choice([1, 1, 2, 3])
            cuts = sorted(rng.randint(0, rows) for _ in range(groups - 1))
            sizes = [b - a for a, b in zip([0] + cuts, cuts + [rows])]
            case.update(rows="+".join(str(n) for n in sizes), batch=batch, tail=rng.choice([0, 0, 1, 77]))
        case.update(inputs=_width(rng), outputs=_width(rng),
                    # a training case has an activation with a continuous derivative: at relu's border another order of the
                    # same sum decides between a gradient and none
                    act=rng.choice(["none", "gelu", "gelu_tanh", "silu"] + (["relu"] if case["mode"] == "infer" else [])),
                    bias=rng.random() < 0.8, residual=rng.random() < 0.4, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
        groups = 1 if case["op"] == "linear" else len(_sizes(case))
        total = _total_rows(case)
        if (total * case["inputs"] * case["outputs"] <= MAX_PRODUCTS and total * max(case["inputs"], case["outputs"]) <= MAX_ELEMENTS
                and groups * case["inputs"] * case["outputs"] <= MAX_ELEMENTS):
            return case


def _sizes(case):
    return [int(v) for v in case["rows"].split("+")]


def _total_rows(case):
    """All rows of x, those of no group among them."""
    if case["op"] == "linear":
        return case["rows"]
    return case["batch"] * (sum(_sizes(case)) + case["tail"])


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    K, N = case["inputs"], case["outputs"]

    def normal(shape, scale=1.0):
        # in slices: the 32-bit numbers of a large tensor are never all there at once
        out = torch.empty(shape, dtype=dt, device=DEVICE)
        flat = out.view(-1)
        for i in range(0, flat.numel(), 1 << 26):
            part = flat[i:i + (1 << 26)]
            part.copy_(torch.randn(part.numel(), generator=gen, device=DEVICE) * scale)
        return out

    if case["op"] == "linear":
        lead, groups, sizes, starts = (case["rows"],), (), None, None
    else:
        sizes = _sizes(case)
        lead, groups = (case["batch"], sum(sizes) + case["tail"]), (len(sizes),)
        starts = torch.tensor([sum(sizes[:i]) for i in range(len(sizes) + (1 if case["tail"] else 0))], dtype=torch.int64, device=DEVICE)
    state = dict(case=case, sizes=sizes, starts=starts)
    state["x"] = normal((*lead, K))                                   # tokens behind a norm
    state["weight"] = normal((*groups, N, K), math.sqrt(2.0 / (K + N)))   # the layers' initial spread
    state["bias"] = normal((*groups, N), 0.1) if case["bias"] else None
    state["residual"] = normal((*lead, N)) if case["residual"] else None
    state["grad"] = normal((*lead, N)) if case["mode"] == "train" else None
    if own and case["mode"] == "train":
        for name in ("x", "weight", "bias", "residual"):
            if state[name] is not None:
                state[name].requires_grad_(True)
    return state


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from ops3d_b200 import fused_linear, grouped_linear

    case = state["case"]
    x, weight, bias, residual = state["x"], state["weight"], state["bias"], state["residual"]
    if case["op"] == "linear":
        y = fused_linear(x, weight, bias, residual=residual, activation=case["act"])
    else:
        y = grouped_linear(x, weight, state["starts"], bias, residual=residual, activation=case["act"])
    if case["mode"] == "infer":
        return y
    names = [n for n in ("x", "weight", "bias", "residual") if state[n] is not None]
    grads = torch.autograd.grad(y, [state[n] for n in names], state["grad"])
    return dict(y=y.detach(), **{"grad_" + n: g for n, g in zip(names, grads)})


def _activate(pre, act):
    if act == "relu":
        return pre.clamp_min(0)
    if act == "gelu":
        return 0.5 * pre * (1 + torch.erf(pre * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * pre * (1 + torch.tanh(math.sqrt(2 / math.pi) * (pre + 0.044715 * pre * pre * pre)))
    if act == "silu":
        return pre * torch.sigmoid(pre)
    return pre


def _slope(pre, act):
    if act == "relu":
        return (pre > 0).to(pre.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(pre * math.sqrt(0.5))) + pre * torch.exp(-0.5 * pre * pre) * (1 / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (pre + 0.044715 * pre * pre * pre))
        return 0.5 * (1 + t) + 0.5 * pre * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * pre * pre)
    s = torch.sigmoid(pre)
    return s * (1 + pre * (1 - s))


def _plain_product(x, weight, bias, grad, act):
    """One weight's product over rows in 32 bits: act(pre), and with ``grad`` the gradients too."""
    pre = x @ weight.t()
    if bias is not None:
        pre = pre + bias
    y = _activate(pre, act)
    if grad is None:
        return y, None, None, None
    g = grad if act == "none" else grad * _slope(pre, act)
    return y, g @ weight, g.t() @ x, None if bias is None else g.sum(0)


def _run_plain(state):
    case = state["case"]
    dt, train = DTYPES[case["dtype"]], case["mode"] == "train"
    x, weight = state["x"].float(), state["weight"].float()
    bias = None if state["bias"] is None else state["bias"].float()
    grad = state["grad"].float() if train else None
    if case["op"] == "linear":
        y, gx, gw, gb = _plain_product(x, weight, bias, grad, case["act"])
    else:
        y = x.new_zeros(*x.shape[:2], case["outputs"])
        if train:
            gx, gw = torch.zeros_like(x), torch.zeros_like(weight)
            gb = None if bias is None else torch.zeros_like(bias)
        begin = 0
        for e, n in enumerate(state["sizes"]):
            if n:
                part = slice(begin, begin + n)
                yg, xg, wg, bg = _plain_product(x[:, part].reshape(-1, case["inputs"]), weight[e], None if bias is None else bias[e],
                                                grad[:, part].reshape(-1, case["outputs"]) if train else None, case["act"])
                y[:, part] = yg.view(case["batch"], n, -1)
                if train:
                    gx[:, part] = xg.view(case["batch"], n, -1)
                    gw[e] = wg
                    if gb is not None:
                        gb[e] = bg
            begin += n
    if state["residual"] is not None:
        y = y + state["residual"].float()
    if not train:
        return y.to(dt)
    out = dict(y=y.to(dt), grad_x=gx.to(dt), grad_weight=gw.to(dt))
    if bias is not None:
        out["grad_bias"] = gb.to(dt)
    if state["residual"] is not None:
        out["grad_residual"] = state["grad"]
    return out


# ---------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    tensors = {k: (v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v) for k, v in state.items()}
    x, w, b, r, dy = (tensors[k] for k in ("x", "weight", "bias", "residual", "grad"))
    K, N = case["inputs"], case["outputs"]
    rows = x.reshape(-1, K)
    if case["op"] == "linear":
        index = [torch.arange(rows.shape[0], device=rows.device)]
        w, b = w[None], None if b is None else b[None]
    else:
        # the rows of each group, over all batch elements
        length, index, begin = x.shape[1], [], 0
        base = torch.arange(case["batch"], device=rows.device)[:, None] * length
        for n in _sizes(case):
            index.append((base + torch.arange(begin, begin + n, device=rows.device)).reshape(-1))
            begin += n
    y = torch.zeros(rows.shape[0], N, dtype=torch.float64, device=rows.device) if r is None else r.reshape(-1, N).clone()
    dx = torch.zeros_like(rows)
    dw, db = torch.zeros_like(w), None if b is None else torch.zeros_like(b)
    for e, all_rows in enumerate(index):
        for some in all_rows.split(1 << 17):
            if some.numel() == 0:
                continue
            z = torch.einsum("mk,nk->mn", rows[some], w[e])
            if b is not None:
                z += b[e]
            phi = torch.special.ndtr(z) if case["act"] == "gelu" else None
            if case["act"] == "none":
                f, slope = z, torch.ones_like(z)
            elif case["act"] == "relu":
                f, slope = torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).double()
            elif case["act"] == "gelu":
                f, slope = z * phi, phi + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
            elif case["act"] == "gelu_tanh":
                c = math.sqrt(2 / math.pi)
                th = torch.tanh(c * z + c * 0.044715 * z ** 3)
                f, slope = z * (1 + th) / 2, (1 + th) / 2 + z / 2 * (1 - th ** 2) * (c + 3 * c * 0.044715 * z ** 2)
            else:
                s = 1 / (1 + torch.exp(-z))
                f, slope = z * s, s + z * s * (1 - s)
            y[some] += f
            if dy is not None:
                g = dy.reshape(-1, N)[some] * slope
                dx[some] = torch.einsum("mn,nk->mk", g, w[e])
                dw[e] += torch.einsum("mn,mk->nk", g, rows[some])
                if db is not None:
                    db[e] += g.sum(0)
    y = y.view(*x.shape[:-1], N)
    if dy is None:
        return y
    out = dict(y=y, grad_x=dx.view_as(x), grad_weight=dw[0] if case["op"] == "linear" else dw)
    if db is not None:
        out["grad_bias"] = db[0] if case["op"] == "linear" else db
    if r is not None:
        out["grad_residual"] = dy
    return out


# ---------------------------------------------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    """Bytes: x, weights, bias, residual and dy read once, y and the gradients written once (dresidual is dy); weights of empty
    groups are not read.  Operations: one product forward, two more in training."""
    K, N, s = case["inputs"], case["outputs"], SIZE[case["dtype"]]
    rows, total = (case["rows"],) * 2 if case["op"] == "linear" else (case["batch"] * sum(_sizes(case)), _total_rows(case))
    groups = used = 1
    if case["op"] == "grouped":
        groups, used = len(_sizes(case)), sum(1 for n in _sizes(case) if n)
    weight = N * K + (N if case["bias"] else 0)
    elements = rows * K + used * weight + total * N + (total * N if case["residual"] else 0)
    flops = 2.0 * rows * N * K
    if case["mode"] == "train":
        elements += rows * N + total * K + groups * weight
        flops *= 3
    return {"bytes": float(elements * s), "flops": flops}
