"""Workloads of the operators of heads whose parts depend on a row's element, dataset or token: which sizes, types and directions,
how their inputs are made, and what a pass through each cannot do without.

  embed   rows of a table by index, scaled, and the table's gradient (rows: atoms or tokens; -1: no entry)
  group   a product with a matrix and a bias of the row's own group (rows in any order, groups of any size, empty ones among
          them; -1: no group).  Forward, and the gradient of x, weights and biases
  clip    the norm of the gradients of many tensors together, and the gradients brought to a norm at most as large as given

`own` false: elementary torch operations in single precision.  `own` true: symmetrix_amd.finetune."""
from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}


def _embed(direction, rows, entries, dim, dtype, scale=1.0):
    return {"op": "embed", "direction": direction, "rows": rows, "entries": entries, "dim": dim, "dtype": dtype, "scale": scale}


def _group(direction, rows, d_in, d_out, groups, dtype, order="mixed"):
    return {"op": "group", "direction": direction, "rows": rows, "d_in": d_in, "d_out": d_out, "groups": groups, "dtype": dtype,
            "order": order}


def _clip(direction, tensors, numel, dtype, packed=False):
    return {"op": "clip", "direction": direction, "tensors": tensors, "numel": numel, "dtype": dtype, "packed": packed}


def listed():
    return [
        # the elements of one small cell: nothing but latency
        dict(_embed("forward", 24, 10, 192, "float32"), name="embed_forward_24"),
        # a long batch of tokens from a large table in 16 bits
        dict(_embed("forward", 32749, 100_003, 4096, "bfloat16", scale=64.0), name="embed_forward_32749_bf16"),
        # training on 50 000 atoms of 89 elements (128 channels, both layers): few entries, long sums
        dict(_embed("gradient", 50000, 89, 256, "float32"), name="embed_gradient_50000"),
        # training on tokens of a large table: most sums short, a few long
        dict(_embed("gradient", 16381, 32000, 2048, "bfloat16", scale=45.25), name="embed_gradient_16381_bf16"),
        # one small cell through a layer of each element's own
        dict(_group("forward", 24, 192, 128, 3, "float32"), name="group_forward_24"),
        # single tokens, nearly every one with another group: weights are read, little is computed
        dict(_group("forward", 48, 2048, 2048, 64, "bfloat16"), name="group_forward_48_bf16"),
        # 3 000 atoms of 10 elements
        dict(_group("forward", 3000, 256, 512, 10, "float32"), name="group_forward_3000"),
        # a large batch through wide layers
        dict(_group("forward", 16381, 4096, 2048, 16, "bfloat16"), name="group_forward_16381_bf16"),
        # a training step's gradient on 50 000 atoms, those of an element one after the other
        dict(_group("gradient", 50000, 256, 512, 12, "float32", order="runs"), name="group_gradient_50000"),
        # the gradient of wide layers
        dict(_group("gradient", 8179, 2048, 2048, 8, "float16"), name="group_gradient_8179_f16"),
        # the norm of one head's gradients
        dict(_clip("norm", 9, 200_003, "float32"), name="norm_head"),
        # a whole model's gradients, clipped
        dict(_clip("clip", 48, 150_000_000, "bfloat16"), name="clip_150m_bf16"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _width(rng, low, high):
    """A multiple of 32 (of 160 for wide rows), or an odd number."""
    d = _spread(rng, low, high)
    step = 32 if d < 1024 else 160
    return max(step, d // step * step) if rng.random() < 0.7 else d | 1


def draw(rng):
    op = rng.choice(["embed", "group", "group", "clip"])
    dtype = rng.choice(list(TYPES))
    if op == "embed":
        dim = _width(rng, 16, 4096)
        direction = rng.choice(["forward", "gradient"])
        rows, entries = _spread(rng, 1, min(65536, 60_000_000 // dim)), _spread(rng, 2, min(200_000, 120_000_000 // dim))
        return _embed(direction, rows, entries, dim, dtype, rng.choice([1.0, math.sqrt(dim), 0.125]))
    if op == "group":
        d_in, d_out, groups = _width(rng, 32, 4096), _width(rng, 32, 4096), _spread(rng, 1, 64)
        groups = max(1, min(groups, 250_000_000 // (d_in * d_out)))
        direction = rng.choice(["forward", "forward", "gradient"])
        # (what a row costs in single precision is more than in 16 bits, in a gradient twice)
        most = int((30e9 if dtype == "float32" else 120e9) / (2 * d_in * d_out))
        return _group(direction, _spread(rng, 1, max(1, min(65536, most))), d_in, d_out, groups, dtype, rng.choice(["mixed", "runs"]))
    return _clip(rng.choice(["norm", "clip"]), _spread(rng, 1, 300), _spread(rng, 2000, 100_000_000), dtype, rng.random() < 0.3)


# ---- inputs

def _sizes(case):
    """Sizes of the tensors: most of the numbers in a few of them, odd ones, single numbers among the small ones."""
    rng = random.Random(case["tensors"] * 1_000_003 + case["numel"])
    weight = [math.exp(rng.uniform(0.0, 6.0)) for _ in range(case["tensors"])]
    total = sum(weight)
    return [max(1, int(case["numel"] * w / total)) for w in weight]


def prepare(case, seed):
    device = torch.device("cuda:0")
    gen = torch.Generator(device=device).manual_seed(seed)
    rng = random.Random(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dtype):
        return torch.randn(*shape, generator=gen, device=device, dtype=torch.float32).mul_(scale).to(dtype)

    if case["op"] == "embed":
        rows, entries, dim = case["rows"], case["entries"], case["dim"]
        # frequent entries and rare ones, as elements and tokens are; one row in sixteen without one
        index = (torch.rand(rows, generator=gen, device=device, dtype=torch.float64) ** 3 * entries).long().clamp_(max=entries - 1)
        index = torch.randperm(entries, generator=gen, device=device)[index].to(torch.int32)
        index[torch.rand(rows, generator=gen, device=device) < 0.0625] = -1
        state = {"case": case, "index": index}
        if case["direction"] == "forward":
            state["table"] = normal(entries, dim, scale=0.05)
        else:
            state["dy"] = normal(rows, dim, scale=1e-2)
        return state
    if case["op"] == "group":
        rows, d_in, d_out, n = case["rows"], case["d_in"], case["d_out"], case["groups"]
        # groups of different sizes, one row in 32 without one
        share = torch.tensor([math.exp(rng.gauss(0.0, 0.7)) for _ in range(n)], device=device)
        index = torch.multinomial(share, rows, replacement=True, generator=gen).to(torch.int32)
        index[torch.rand(rows, generator=gen, device=device) < 0.03125] = -1
        if case["order"] == "runs":
            index = torch.sort(index).values
        state = {"case": case, "index": index, "x": normal(rows, d_in), "weight": normal(n, d_out, d_in, scale=d_in ** -0.5)}
        if case["direction"] == "forward":
            state["bias"] = normal(n, d_out, scale=0.1)
        else:
            state["dy"] = normal(rows, d_out)
        return state

    # Gradients lie in one array, a tensor starting at a multiple of 256 numbers, or, packed, right behind the one before it.
    sizes, pad = _sizes(case), 1 if case["packed"] else 256
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += -(-n // pad) * pad
    grad = torch.zeros(at, dtype=dtype, device=device)
    for b, n in zip(starts, sizes):
        grad[b:b + n] = normal(n, scale=1e-2 * math.exp(rng.gauss(0.0, 1.0)))
    state = {"case": case, "grads": [grad[b:b + n] for b, n in zip(starts, sizes)]}
    if case["direction"] == "clip":
        # (a tenth to a half of what the norm is)
        state["max_norm"] = rng.uniform(0.1, 0.5) * 1e-2 * math.sqrt(sum(sizes))
        state["clipped"] = torch.zeros_like(grad)
        state["out"] = [state["clipped"][b:b + n] for b, n in zip(starts, sizes)]
    return state


# ---- the plain forms

def _plain_embed(s):
    case, index = s["case"], s["index"].long()
    if case["direction"] == "forward":
        y = s["table"][index.clamp(min=0)].float() * case["scale"]
        return {"y": torch.where((index >= 0)[:, None], y, torch.zeros_like(y)).to(s["table"].dtype)}
    # (rows without an entry go to one behind the last)
    n = case["entries"]
    sums = torch.zeros(n + 1, case["dim"], device=index.device).index_add_(0, torch.where(index >= 0, index, n), s["dy"].float())
    return {"dtable": (sums[:n] * case["scale"]).to(s["dy"].dtype)}


def _plain_group(s):
    case, index, dtype = s["case"], s["index"].long(), s["x"].dtype
    n = case["groups"]
    order = torch.argsort(index, stable=True)
    counts = torch.bincount(index + 1, minlength=n + 1).tolist()
    forward = case["direction"] == "forward"
    if forward:
        y = torch.zeros(case["rows"], case["d_out"], device=index.device, dtype=dtype)
    else:
        dx = torch.zeros_like(s["x"])
        dw = torch.zeros_like(s["weight"])
        db = torch.zeros(n, case["d_out"], device=index.device, dtype=dtype)
    end = counts[0]
    for k in range(n):
        begin, end = end, end + counts[k + 1]
        if begin == end:
            continue
        at = order[begin:end]
        w = s["weight"][k].float()
        if forward:
            y[at] = (s["x"][at].float() @ w.t() + s["bias"][k].float()).to(dtype)
        else:
            dy = s["dy"][at].float()
            dx[at] = (dy @ w).to(dtype)
            dw[k] = (dy.t() @ s["x"][at].float()).to(dtype)
            db[k] = dy.sum(0).to(dtype)
    return {"y": y} if forward else {"dx": dx, "dweight": dw, "dbias": db}


def _plain_clip(s):
    norm = torch.stack([g.float().square().sum().double() for g in s["grads"]]).sum().sqrt().float()
    if s["case"]["direction"] == "norm":
        return {"norm": norm}
    factor = torch.clamp(s["max_norm"] / norm, max=1.0)
    for g, o in zip(s["grads"], s["out"]):
        o.copy_(g.float() * factor)
    return {"norm": norm, "clipped": s["clipped"]}


# ---- the framework's operators

def _own(s):
    from symmetrix_amd import finetune
    case = s["case"]
    if case["op"] == "embed":
        if case["direction"] == "forward":
            return {"y": finetune.embedding_forward(s["table"], s["index"], case["scale"])}
        return {"dtable": finetune.embedding_backward(s["dy"], s["index"], case["entries"], case["scale"])}
    if case["op"] == "group":
        if case["direction"] == "forward":
            return {"y": finetune.grouped_linear_forward(s["x"], s["weight"], s["bias"], s["index"])}
        dx, dw, db = finetune.grouped_linear_backward(s["dy"], s["x"], s["weight"], s["index"])
        return {"dx": dx, "dweight": dw, "dbias": db}
    if case["direction"] == "norm":
        return {"norm": finetune.grad_norm(s["grads"])}
    return {"norm": finetune.clip_grads(s["grads"], s["max_norm"], out=s["out"]), "clipped": s["clipped"]}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"embed": _plain_embed, "group": _plain_group, "clip": _plain_clip}[state["case"]["op"]](state)


# ---- what a pass cannot do without

def _distinct(case):
    """Entries that occur among a case's rows, as many as are to be expected."""
    rows, n = case["rows"] * 0.9375, case["entries"]
    edges = [(e / n) ** (1 / 3) for e in range(n + 1)]
    return sum(-math.expm1(rows * math.log1p(edges[e] - edges[e + 1])) for e in range(1, n)) + 1


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "embed":
        rows, entries, dim = case["rows"], case["entries"], case["dim"]
        if case["direction"] == "forward":
            return {"bytes": size * dim * (rows + int(_distinct(case))) + 4 * rows, "flops": rows * dim}
        return {"bytes": size * dim * (rows + entries) + 4 * rows, "flops": rows * dim}
    if case["op"] == "group":
        rows, d_in, d_out, n = case["rows"], case["d_in"], case["d_out"], case["groups"]
        if case["direction"] == "forward":
            return {"bytes": size * (rows * (d_in + d_out) + min(n, rows) * (d_in + 1) * d_out) + 4 * rows, "flops": 2 * rows * d_in * d_out}
        return {"bytes": size * (rows * (2 * d_in + d_out) + min(n, rows) * d_in * d_out + n * (d_in + 1) * d_out) + 4 * rows,
                "flops": 4 * rows * d_in * d_out}
    numel = sum(_sizes(case))
    if case["direction"] == "norm":
        return {"bytes": size * numel + 4, "flops": 2 * numel}
    return {"bytes": 2 * size * numel + 4, "flops": 3 * numel}


# ---- in 64 bits, from the definitions

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed":
        index, n, scale = s["index"].long(), case["entries"], case["scale"]
        has = (index >= 0).nonzero()[:, 0]
        if case["direction"] == "forward":
            y = torch.zeros(case["rows"], case["dim"], device=index.device, dtype=torch.float64)
            y[has] = s["table"].double().index_select(0, index[has]) * scale
            return {"y": y}
        order = has[torch.argsort(index[has], stable=True)]
        out = torch.zeros(n, case["dim"], device=index.device, dtype=torch.float64)
        # (the sums of neighbours in sorted order are differences of their running sums, a part of the columns at a time)
        ends = torch.searchsorted(index[order], torch.arange(n, device=index.device), right=True)
        for c in range(0, case["dim"], 256):
            run_sums = torch.cumsum(s["dy"][:, c:c + 256].index_select(0, order).double(), 0)
            run_sums = torch.cat([torch.zeros_like(run_sums[:1]) if len(run_sums) else torch.zeros(1, min(256, case["dim"] - c), device=index.device, dtype=torch.float64), run_sums])
            out[:, c:c + 256] = scale * torch.diff(run_sums[ends], dim=0, prepend=torch.zeros_like(run_sums[:1]))
        return {"dtable": out}
    if case["op"] == "group":
        rows_of = {}
        for i, k in enumerate(s["index"].tolist()):
            rows_of.setdefault(k, []).append(i)
        device, n = s["x"].device, case["groups"]
        if case["direction"] == "forward":
            out = {"y": torch.zeros(case["rows"], case["d_out"], device=device, dtype=torch.float64)}
        else:
            out = {"dx": torch.zeros_like(s["x"], dtype=torch.float64), "dweight": torch.zeros_like(s["weight"], dtype=torch.float64),
                   "dbias": torch.zeros(n, case["d_out"], device=device, dtype=torch.float64)}
        for k, rows in rows_of.items():
            if k < 0:
                continue
            at = torch.tensor(rows, device=device)
            x, w = s["x"].index_select(0, at).double(), s["weight"][k].double()
            if case["direction"] == "forward":
                out["y"].index_copy_(0, at, torch.addmm(s["bias"][k].double(), x, w.t()))
            else:
                dy = s["dy"].index_select(0, at).double()
                out["dx"].index_copy_(0, at, torch.mm(dy, w))
                out["dweight"][k] = torch.mm(x.t(), dy).t()
                out["dbias"][k] = torch.mv(dy.t(), torch.ones(len(rows), device=device, dtype=torch.float64))
        return out
    norm = math.sqrt(math.fsum(float(torch.dot(g.double(), g.double())) for g in s["grads"]))
    value = torch.tensor(norm, device=s["grads"][0].device, dtype=torch.float64)
    if case["direction"] == "norm":
        return {"norm": value}
    for g, o in zip(s["grads"], s["out"]):
        o.copy_(g)
    return {"norm": value, "clipped": s["clipped"].double() * min(1.0, s["max_norm"] / norm)}
