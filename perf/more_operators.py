"""Performance cases of what stands around the products of a transformer layer with experts: layer norm of a residual sum, the
choice of experts for each token, the rows sorted by expert (``grouped_linear`` takes them so) and their weighted sums per token.

    layer_norm      s = x + residual,  y = (s - mean(s)) / sqrt(var(s) + eps) * weight + bias, per row
    route_experts   score = softmax(logits) or sigmoid(logits); the top_k largest of score + bias, inside the top_groups best groups;
                    weight = scale * score / sum of the chosen scores (or scale * score)
    dispatch_rows   the row of x for each (token, choice), sorted by expert, in the order of the tokens within one
    combine_rows    y[token] = sum of weight * row over the token's choices + residual

``listed()`` holds named cases, ``draw(rng)`` further ones of the same ranges; ``prepare`` builds what a program has in hand
before the call, ``run`` is one pass (``own``: through this package, else in elementary torch operations), ``exact`` the same
from the definition in 64 bits, ``work`` the bytes and operations that a pass cannot do without.

A case is a dict of plain values.  ``mode`` "train" is the forward and the gradients of everything that has one.  Ties between
experts go to the lowest index; an expert of -1 (a padded token) belongs to none.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5

# What a drawn case may cost at most: the largest listed one's elements.
MAX_NORM = 598016 * 256
MAX_ROUTE = 149504 * 256
MAX_ROWS = 149504 * 4 * 256


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # One token of a stream behind an attention layer: latency of a single call.
        dict(name="norm one token bf16 infer", op="norm", mode="infer", rows=1, width=256, dtype="bf16", params="same",
             residual="same", keep_sum=False),
        # 200 object queries of four images, training in half precision around an fp32 stream that goes on behind the norm.
        dict(name="norm decoder queries f16 train", op="norm", mode="train", rows=800, width=256, dtype="f16", params="f32",
             residual="f32", keep_sum=True),
        # Features with three coordinates appended: rows that no vector divides.
        dict(name="norm odd width f32 train", op="norm", mode="train", rows=9473, width=259, dtype="f32", params="same",
             residual="none", keep_sum=False),
        # The hidden rows of a feed-forward over one pyramid of 73 728 cells.
        dict(name="norm hidden rows f16 infer", op="norm", mode="infer", rows=73728, width=1024, dtype="f16", params="same",
             residual="none", keep_sum=False),
        # Post-norm of an encoder layer over one tile of 598 016 cells.
        dict(name="norm encoder bf16 train", op="norm", mode="train", rows=598016, width=256, dtype="bf16", params="f32",
             residual="same", keep_sum=False),
        # One token's choice of 2 out of 24 experts.
        dict(name="route one token f32 infer", op="route", mode="infer", tokens=1, experts=24, top_k=2, score="softmax",
             biased=False, groups=1, top_groups=1, group_score="max", renormalise=True, scale=1.0, dtype="f32"),
        # Sigmoid scores with a bias for balance, 3 of 8 groups, over a pyramid of 37 376 cells.
        dict(name="route grouped bf16 infer", op="route", mode="infer", tokens=37376, experts=64, top_k=6, score="sigmoid",
             biased=True, groups=8, top_groups=3, group_score="top2", renormalise=True, scale=2.5, dtype="bf16"),
        # Four such pyramids, 8 of 256 experts, training.
        dict(name="route many experts bf16 train", op="route", mode="train", tokens=149504, experts=256, top_k=8,
             score="softmax", biased=True, groups=1, top_groups=1, group_score="max", renormalise=True, scale=1.0, dtype="bf16"),
        # A handful of tokens to their experts.
        dict(name="dispatch tokens bf16 infer", op="dispatch", mode="infer", tokens=4, experts=24, top_k=2, width=256,
             padded=0.0, dtype="bf16"),
        # 73 728 cells to 16 experts, some of them padding, training.
        dict(name="dispatch cells f16 train", op="dispatch", mode="train", tokens=73728, experts=16, top_k=2, width=256,
             padded=0.05, dtype="f16"),
        # The experts' results of 3001 tokens, rows that no vector divides.
        dict(name="combine odd width f32 infer", op="combine", mode="infer", tokens=3001, experts=131, top_k=3, width=99,
             padded=0.1, weighted=True, residual=True, dtype="f32"),
        # The results of four experts per cell over four pyramids of 37 376 cells, training.
        dict(name="combine cells bf16 train", op="combine", mode="train", tokens=149504, experts=64, top_k=4, width=256,
             padded=0.0, weighted=True, residual=True, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, most):
    """A feature width: mostly a multiple of 8, as layers have them, sometimes any number."""
    n = _log_int(rng, 8, most)
    return n if rng.random() < 0.25 else max(8, n // 8 * 8)


def draw(rng):
    op = rng.choice(["norm", "route", "dispatch", "combine"])
    case = dict(op=op, mode=rng.choice(["infer", "train"]))
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    while True:
        tokens = 1 if rng.random() < 0.08 else _log_int(rng, 1, 600000 if op == "norm" else 150000)
        experts = _log_int(rng, 4, 512)
        if op == "norm":
            width = _width(rng, 8192)
            if tokens * width > MAX_NORM:
                continue
            residual = rng.choice(["none", "same", "same"] + (["f32"] if dtype != "f32" else []))
            case.update(rows=tokens, width=width, dtype=dtype, params=rng.choice(["same", "f32"]), residual=residual,
                        keep_sum=residual != "none" and rng.random() < 0.5)
        elif op == "route":
            if tokens * experts > MAX_ROUTE:
                continue
            groups = rng.choice([1, 1, 2, 4, 8])
            experts = max(1, experts // groups) * groups
            top_groups = rng.randint(1, groups)
            top_k = rng.randint(1, min(16, top_groups * (experts // groups)))
            case.update(tokens=tokens, experts=experts, top_k=top_k, score=rng.choice(["softmax", "sigmoid"]),
                        biased=rng.random() < 0.6, groups=groups, top_groups=top_groups, group_score=rng.choice(["max", "top2"]),
                        renormalise=top_k > 1 and rng.random() < 0.6, scale=rng.choice([1.0, 2.5]), dtype=dtype)
        else:
            width, top_k = _width(rng, 4096), rng.randint(1, min(8, experts))
            if tokens * top_k * width > MAX_ROWS:
                continue
            case.update(tokens=tokens, experts=experts, top_k=top_k, width=width, padded=rng.choice([0.0, 0.0, 0.1, 0.5]))
            if op == "combine":
                case.update(weighted=rng.random() < 0.8, residual=rng.random() < 0.5)
            case["dtype"] = dtype
        return case


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    train = case["mode"] == "train"

    def normal(shape, scale=1.0, mean=0.0, dtype=dt):
        # in slices: the 32-bit numbers of a large tensor are never all there at once
        out = torch.empty(shape, dtype=dtype, device=DEVICE)
        flat = out.view(-1)
        for i in range(0, flat.numel(), 1 << 26):
            part = flat[i:i + (1 << 26)]
            part.copy_(torch.randn(part.numel(), generator=gen, device=DEVICE) * scale + mean)
        return out

    state = dict(case=case)
    if case["op"] == "norm":
        shape, C = (case["rows"], case["width"]), case["width"]
        pdt = dt if case["params"] == "same" else torch.float32
        rdt = dt if case["residual"] == "same" else torch.float32
        state["x"] = normal(shape)
        state["weight"], state["bias"] = normal((C,), 0.1, 1.0, pdt), normal((C,), 0.1, 0.0, pdt)
        # a stream that has grown over some layers, with a mean of its own
        state["residual"] = None if case["residual"] == "none" else normal(shape, 2.0, 0.3, rdt)
        state["grad"] = normal(shape) if train else None
        state["grad_sum"] = normal(shape, 1.0, 0.0, rdt) if train and case["keep_sum"] else None
        leaves = ("x", "weight", "bias", "residual")
    elif case["op"] == "route":
        T, E, k = case["tokens"], case["experts"], case["top_k"]
        state["logits"] = normal((T, E), 1.5)
        state["bias"] = normal((E,), 0.02, 0.0, torch.float32) if case["biased"] else None
        state["grad"] = normal((T, k), 1.0, 0.0, torch.float32) if train else None
        leaves = ("logits",)
    else:
        T, E, k, C = case["tokens"], case["experts"], case["top_k"], case["width"]
        # distinct experts per token, some more popular than others; padded tokens have none
        popular = torch.randn(E, generator=gen, device=DEVICE)
        experts = (torch.randn(T, E, generator=gen, device=DEVICE) + popular).topk(k, -1).indices
        if case["padded"]:
            experts[torch.rand(T, generator=gen, device=DEVICE) < case["padded"]] = -1
        state["experts"] = experts
        if case["op"] == "dispatch":
            state["x"] = normal((T, C))
            state["grad"] = normal((T * k, C)) if train else None
            leaves = ("x",)
        else:
            state["rows"] = normal((T * k, C))
            state["weights"] = torch.rand(T, k, generator=gen, device=DEVICE) if case["weighted"] else None
            state["residual"] = normal((T, C)) if case["residual"] else None
            state["grad"] = normal((T, C)) if train else None
            leaves = ("rows", "weights", "residual")
            # the order that the experts' rows were dispatched in
            if own:
                from ops3d_b200 import dispatch_rows

                state["order"] = dispatch_rows(torch.empty(T, 1, dtype=dt, device=DEVICE), experts, E)[1]
            else:
                state["starts"], state["position"] = _order(experts, E)
    state["leaves"] = [name for name in leaves if state[name] is not None]
    if own and train:
        for name in state["leaves"]:
            state[name].requires_grad_(True)
    return state


def _order(experts, n_experts):
    """Start of each expert's rows (and the end of the last one's), and where the row of each choice stands; -1 for none."""
    flat = experts.reshape(-1)
    key = torch.where((flat >= 0) & (flat < n_experts), flat, n_experts)
    source = torch.sort(key, stable=True).indices
    position = torch.empty_like(source)
    position[source] = torch.arange(source.numel(), device=source.device)
    counts = torch.zeros(n_experts + 1, dtype=key.dtype, device=key.device).scatter_add_(0, key, torch.ones_like(key))[:n_experts]
    starts = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    return starts, torch.where(key < n_experts, position, -1).view(experts.shape)


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else PLAIN[state["case"]["op"]](state)


def _run_own(state):
    import ops3d_b200 as ops

    case = state["case"]
    if case["op"] == "norm":
        out = ops.layer_norm(state["x"], state["weight"], state["bias"], residual=state["residual"], eps=EPS,
                             return_sum=case["keep_sum"])
        outputs = dict(zip(("y", "sum"), out)) if case["keep_sum"] else dict(y=out)
        grads = [state["grad"], state["grad_sum"]][:len(outputs)]
        differentiable = list(outputs.values())
    elif case["op"] == "route":
        weights, experts = ops.route_experts(state["logits"], case["top_k"], bias=state["bias"], score=case["score"],
                                             n_groups=case["groups"], top_groups=case["top_groups"], group_score=case["group_score"],
                                             renormalise=case["renormalise"], scale=case["scale"])
        outputs, differentiable, grads = dict(weights=weights, experts=experts), [weights], [state["grad"]]
    elif case["op"] == "dispatch":
        rows, order = ops.dispatch_rows(state["x"], state["experts"], case["experts"])
        outputs = dict(rows=rows, starts=order.group_start_index, position=order.position)
        differentiable, grads = [rows], [state["grad"]]
    else:
        y = ops.combine_rows(state["rows"], state["order"], state["weights"], residual=state["residual"])
        outputs, differentiable, grads = dict(y=y), [y], [state["grad"]]
    if case["mode"] == "train":
        back = torch.autograd.grad(differentiable, [state[name] for name in state["leaves"]], grads)
        outputs = {name: t.detach() for name, t in outputs.items()}
        outputs.update(("grad_" + name, g) for name, g in zip(state["leaves"], back))
    return outputs


def _plain_norm(state):
    case = state["case"]
    x, w, b = state["x"].float(), state["weight"].float(), state["bias"].float()
    s = x if state["residual"] is None else x + state["residual"].float()
    centred = s - s.mean(-1, keepdim=True)
    inverse = 1 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    unit = centred * inverse
    out = dict(y=(unit * w + b).to(state["x"].dtype))
    if case["keep_sum"]:
        out["sum"] = s.to(state["residual"].dtype)
    if case["mode"] == "infer":
        return out
    dy = state["grad"].float()
    g = dy * w
    ds = inverse * (g - g.mean(-1, keepdim=True) - unit * (g * unit).mean(-1, keepdim=True))
    if case["keep_sum"]:
        ds = ds + state["grad_sum"].float()
    out["grad_x"] = ds.to(state["x"].dtype)
    out["grad_weight"] = (dy * unit).sum(0).to(state["weight"].dtype)
    out["grad_bias"] = dy.sum(0).to(state["bias"].dtype)
    if state["residual"] is not None:
        out["grad_residual"] = ds.to(state["residual"].dtype)
    return out


def _plain_route(state):
    case, T, E = state["case"], state["case"]["tokens"], state["case"]["experts"]
    # which experts: in 64 bits, because scores next to one another decide
    logits = state["logits"].double()
    if case["score"] == "softmax":
        shifted = torch.exp(logits - logits.max(-1, keepdim=True).values)
        score = shifted / shifted.sum(-1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-logits))
    select = score if state["bias"] is None else score + state["bias"].double()
    if case["groups"] > 1:
        each = torch.sort(select.view(T, case["groups"], -1), dim=-1, descending=True).values
        value = each[..., 0] if case["group_score"] == "max" or each.shape[-1] == 1 else each[..., 0] + each[..., 1]
        best = torch.sort(value, dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        allowed = torch.zeros_like(value, dtype=torch.bool).scatter_(1, best, True)
        select = torch.where(allowed.repeat_interleave(E // case["groups"], 1), select, -math.inf)
    experts = torch.sort(select, dim=-1, descending=True, stable=True).indices[:, :case["top_k"]].contiguous()
    # weights and gradients: in 32
    logits = state["logits"].float()
    if case["score"] == "softmax":
        shifted = torch.exp(logits - logits.max(-1, keepdim=True).values)
        score = shifted / shifted.sum(-1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-logits))
    chosen = score.gather(1, experts)
    total = chosen.sum(-1, keepdim=True)
    weights = chosen / total * case["scale"] if case["renormalise"] else chosen * case["scale"]
    out = dict(weights=weights, experts=experts)
    if case["mode"] == "infer":
        return out
    dw = state["grad"] * case["scale"]
    dchosen = (dw - (dw * chosen).sum(-1, keepdim=True) / total) / total if case["renormalise"] else dw
    dscore = torch.zeros_like(score).scatter_(1, experts, dchosen)
    if case["score"] == "softmax":
        dlogits = score * (dscore - (dscore * score).sum(-1, keepdim=True))
    else:
        dlogits = dscore * score * (1 - score)
    out["grad_logits"] = dlogits.to(state["logits"].dtype)
    return out


def _spread(each, flat):
    """Rows at their positions; those of none go to one more row, which is dropped."""
    n = flat.numel()
    rows = torch.zeros(n + 1, each.shape[1], device=each.device)
    rows[torch.where(flat >= 0, flat, n)] = each
    return rows[:n]


def _plain_dispatch(state):
    case, x = state["case"], state["x"]
    starts, position = _order(state["experts"], case["experts"])
    flat = position.reshape(-1)
    rows = _spread(x.float().repeat_interleave(case["top_k"], 0), flat)
    out = dict(rows=rows.to(x.dtype), starts=starts, position=position)
    if case["mode"] == "train":
        here = state["grad"].float()[flat.clamp_min(0)] * (flat >= 0)[:, None]
        out["grad_x"] = here.view(case["tokens"], case["top_k"], -1).sum(1).to(x.dtype)
    return out


def _plain_combine(state):
    case, rows = state["case"], state["rows"]
    flat = state["position"].reshape(-1)
    there = (flat >= 0)[:, None]
    each = (rows.float()[flat.clamp_min(0)] * there).view(case["tokens"], case["top_k"], -1)
    weights = torch.ones(case["tokens"], case["top_k"], device=rows.device) if state["weights"] is None else state["weights"]
    y = (each * weights[..., None]).sum(1)
    if state["residual"] is not None:
        y = y + state["residual"].float()
    out = dict(y=y.to(rows.dtype))
    if case["mode"] == "infer":
        return out
    dy = state["grad"].float()
    spread = (dy[:, None] * weights[..., None]).reshape(flat.numel(), -1)
    out["grad_rows"] = _spread(spread, flat).to(rows.dtype)
    if state["weights"] is not None:
        out["grad_weights"] = (each * dy[:, None]).sum(-1)
    if state["residual"] is not None:
        out["grad_residual"] = state["grad"]
    return out


PLAIN = dict(norm=_plain_norm, route=_plain_route, dispatch=_plain_dispatch, combine=_plain_combine)


# ---------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    return EXACT[case["op"]](case, {n: (t.detach().double() if torch.is_tensor(t) and t.is_floating_point() else t) for n, t in state.items()})


def _exact_norm(case, t):
    x, w, b, r, dy, dsum = (t[n] for n in ("x", "weight", "bias", "residual", "grad", "grad_sum"))
    out = {"y": torch.empty_like(x)}
    if case["keep_sum"]:
        out["sum"] = torch.empty_like(x)
    if dy is not None:
        out.update(grad_x=torch.empty_like(x), grad_weight=torch.zeros_like(w), grad_bias=torch.zeros_like(b))
        if r is not None:
            out["grad_residual"] = out["grad_x"]
    for i in range(0, x.shape[0], 1 << 16):
        part = slice(i, i + (1 << 16))
        s = x[part] if r is None else x[part] + r[part]
        var, mean = torch.var_mean(s, -1, correction=0, keepdim=True)
        sd = (var + EPS).sqrt()
        z = (s - mean) / sd
        out["y"][part] = torch.addcmul(b, z, w)
        if case["keep_sum"]:
            out["sum"][part] = s
        if dy is not None:
            d = dy[part]
            out["grad_weight"] += torch.einsum("rc,rc->c", d, z)
            out["grad_bias"] += d.sum(0)
            # the projection of d * w off the directions of 1 and z
            u = d * w
            along = torch.einsum("rc,rc->r", u, z)[:, None] / case["width"]
            ds = (u - u.mean(-1, keepdim=True) - along * z) / sd
            out["grad_x"][part] = ds if dsum is None else ds + dsum[part]
    return out


def _exact_route(case, t):
    logits, bias, dw = t["logits"], t["bias"], t["grad"]
    T, E, G, k = case["tokens"], case["experts"], case["groups"], case["top_k"]
    score = torch.softmax(logits, -1) if case["score"] == "softmax" else torch.sigmoid(logits)
    select = score.clone() if bias is None else score + bias
    rows = torch.arange(T, device=select.device)
    if G > 1:
        inside = select.view(T, G, E // G).clone()
        first, where = inside.max(-1)                                   # the lowest index of a tie
        value = first
        if case["group_score"] == "top2" and E // G > 1:
            inside.scatter_(2, where[..., None], -math.inf)
            value = first + inside.amax(-1)
        keep = torch.zeros(T, G, dtype=torch.bool, device=select.device)
        for _ in range(case["top_groups"]):
            best = _first_largest(value)
            keep[rows, best] = True
            value[rows, best] = -math.inf
        select = select.view(T, G, E // G).masked_fill(~keep[..., None], -math.inf).view(T, E)
    experts = []
    for _ in range(k):
        best = _first_largest(select)
        experts.append(best)
        select[rows, best] = -math.inf
    experts = torch.stack(experts, 1)
    chosen = score.gather(1, experts)
    norm = chosen.sum(1, keepdim=True) if case["renormalise"] else torch.ones_like(chosen[:, :1])
    weights = case["scale"] * chosen / norm
    out = dict(weights=weights, experts=experts)
    if dw is not None:
        # d weight_j / d score_i = scale (delta_ij - [renormalised] chosen_j / sum) / norm
        back = case["scale"] / norm * dw
        if case["renormalise"]:
            back = back - (dw * weights).sum(1, keepdim=True) / norm
        if case["score"] == "sigmoid":
            grad = torch.zeros_like(score).scatter_(1, experts, back * chosen * (1 - chosen))
        else:
            grad = -score * (back * chosen).sum(1, keepdim=True)
            grad.scatter_add_(1, experts, back * chosen)
        out["grad_logits"] = grad
    return out


def _first_largest(values):
    """Index of the largest value of each row, the lowest where several are equal."""
    top = values.amax(-1, keepdim=True)
    index = torch.arange(values.shape[-1], device=values.device).expand_as(values)
    return torch.where(values == top, index, values.shape[-1]).amin(-1)


def _exact_positions(case, experts):
    """Of each choice: how many choices of lower experts there are, and how many of its own before it."""
    flat = experts.reshape(-1)
    n = flat.numel()
    position = torch.full((n,), -1, dtype=torch.int64, device=flat.device)
    starts = [0]
    for e in range(case["experts"]):
        mine = torch.nonzero(flat == e)[:, 0]
        position[mine] = starts[-1] + torch.arange(mine.numel(), device=flat.device)
        starts.append(starts[-1] + mine.numel())
    return torch.tensor(starts, device=flat.device), position.view(experts.shape)


def _exact_dispatch(case, t):
    x, dr = t["x"], t["grad"]
    starts, position = _exact_positions(case, t["experts"])
    T, k, C = case["tokens"], case["top_k"], case["width"]
    rows = torch.zeros(T * k, C, dtype=x.dtype, device=x.device)
    dx = torch.zeros_like(x)
    for j in range(k):
        token = torch.nonzero(position[:, j] >= 0)[:, 0]
        rows.index_copy_(0, position[token, j], x[token])
        if dr is not None:
            dx[token] += dr[position[token, j]]
    out = dict(rows=rows, starts=starts, position=position)
    if dr is not None:
        out["grad_x"] = dx
    return out


def _exact_combine(case, t):
    rows, weights, residual, dy = (t[n] for n in ("rows", "weights", "residual", "grad"))
    _, position = _exact_positions(case, t["experts"])
    y = torch.zeros(case["tokens"], case["width"], dtype=rows.dtype, device=rows.device) if residual is None else residual.clone()
    drows = torch.zeros_like(rows)
    dweights = None if weights is None else torch.zeros_like(weights)
    for j in range(case["top_k"]):
        token = torch.nonzero(position[:, j] >= 0)[:, 0]
        mine = rows[position[token, j]]
        factor = 1.0 if weights is None else weights[token, j][:, None]
        y[token] += factor * mine
        if dy is not None:
            drows[position[token, j]] = factor * dy[token]
            if weights is not None:
                dweights[token, j] = torch.einsum("rc,rc->r", mine, dy[token])
    out = dict(y=y)
    if dy is not None:
        out["grad_rows"] = drows
        if weights is not None:
            out["grad_weights"] = dweights
        if residual is not None:
            out["grad_residual"] = dy
    return out


EXACT = dict(norm=_exact_norm, route=_exact_route, dispatch=_exact_dispatch, combine=_exact_combine)


# ---------------------------------------------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    """Bytes: every input read once, every output written once (gradients that are equal by definition are one tensor); a few
    operations per element."""
    s, train = SIZE[case["dtype"]], case["mode"] == "train"
    if case["op"] == "norm":
        n, C = case["rows"] * case["width"], case["width"]
        p = s if case["params"] == "same" else 4
        r = {"none": 0, "same": s, "f32": 4}[case["residual"]]
        size = n * (2 * s + r + (r if case["keep_sum"] else 0)) + 2 * C * p
        flops = 8.0 * n
        if train:
            size += n * (2 * s + (r if case["keep_sum"] else 0) + (4 if case["residual"] == "f32" else 0)) + 2 * C * p
            flops += 15.0 * n
    elif case["op"] == "route":
        n, m = case["tokens"] * case["experts"], case["tokens"] * case["top_k"]
        size = n * s + m * 12 + (case["experts"] * 4 if case["biased"] else 0)
        flops = 4.0 * n
        if train:
            size += m * 4 + n * s
            flops += 4.0 * n
    else:
        T, k, C = case["tokens"], case["top_k"], case["width"]
        m = T * k
        if case["op"] == "dispatch":
            size = T * C * s + m * 16 + (case["experts"] + 1) * 8 + m * C * s
            flops = float(m)
            if train:
                size += m * C * s + T * C * s
                flops += m * C
        else:
            w = 4 if case["weighted"] else 0
            size = m * C * s + m * (8 + w) + T * C * s * (2 if case["residual"] else 1)
            flops = 2.0 * m * C
            if train:
                size += T * C * s + m * C * s + m * w
                flops += 3.0 * m * C
    return {"bytes": float(size), "flops": float(flops)}
