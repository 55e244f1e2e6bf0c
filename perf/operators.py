"""Workloads of the operators that fine-tune a head on the engine's atomic descriptors and serve it: which sizes, types and
directions, how their inputs are made, and what a pass through each cannot do without.

  norm    layer norm over the features of an atom (rows: atoms), forward with the rows' statistics, and the gradient of
          features, weight and bias
  adapt   a shared projection with a low-rank adapter per row beside it: rows belong to requests (systems, datasets, users),
          every request has an adapter of its own or none (-1):  y = W x + scale_a B_a (A_a x).  Forward, and the gradient of
          x, A and B with W fixed
  adamw   one AdamW step over many tensors, with moments in 32 bits or in 8 (256 numbers to a scale), and with
          single-precision masters of parameters in 16 bits

`own` false: elementary torch operations in single precision.  `own` true: symmetrix_amd.finetune."""
from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
EPS = 1e-5
BLOCK = 256                    # numbers to a scale of moments in 8 bits
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 1e-2
FIRST_STEP = 10


def _norm(direction, rows, dim, dtype, pitch=1):
    return {"op": "norm", "direction": direction, "rows": rows, "dim": dim, "dtype": dtype, "pitch": pitch}


def _adapt(direction, rows, d_in, d_out, rank, adapters, dtype, single=False):
    return {"op": "adapt", "direction": direction, "rows": rows, "d_in": d_in, "d_out": d_out, "rank": rank,
            "adapters": adapters, "dtype": dtype, "single": single}


def _adamw(tensors, numel, dtype, bits, masters=False, packed=False):
    return {"op": "adamw", "tensors": tensors, "numel": numel, "dtype": dtype, "bits": bits, "masters": masters, "packed": packed}


def listed():
    return [
        # descriptors of one small cell (96 channels, both layers): nothing but latency
        dict(_norm("forward", 24, 192, "float32"), name="norm_forward_24"),
        # long batches of wide rows in 16 bits
        dict(_norm("forward", 16381, 4096, "bfloat16"), name="norm_forward_16381_bf16"),
        # training on the descriptors of 50 000 atoms (128 channels, both layers)
        dict(_norm("gradient", 50000, 256, "float32"), name="norm_gradient_50000"),
        # one small cell through an adapted projection
        dict(_adapt("forward", 24, 192, 128, 4, 3, "float32"), name="adapt_forward_24"),
        # sixteen requests of one row each, every one with another adapter: weights are read, little is computed
        dict(_adapt("forward", 16, 4096, 4096, 16, 64, "bfloat16", single=True), name="adapt_forward_16_single_bf16"),
        # 50 000 atoms of many systems, adapters of a dozen datasets
        dict(_adapt("forward", 50000, 256, 512, 8, 12, "float32"), name="adapt_forward_50000"),
        # a large batch through a wide projection
        dict(_adapt("forward", 8179, 4096, 4096, 32, 24, "bfloat16"), name="adapt_forward_8179_bf16"),
        # a training step's gradient on 20 011 atoms
        dict(_adapt("gradient", 20011, 256, 512, 8, 12, "float32"), name="adapt_gradient_20011"),
        # the gradient of a wide projection's adapters
        dict(_adapt("gradient", 4091, 2048, 2048, 16, 16, "float16"), name="adapt_gradient_4091_f16"),
        # the tensors of one adapted head
        dict(_adamw(9, 200_003, "float32", 32), name="adamw_head"),
        # a whole model in bfloat16 with single-precision masters
        dict(_adamw(48, 150_000_000, "bfloat16", 32, masters=True), name="adamw_150m_bf16"),
        # moments in 8 bits, where memory is short
        dict(_adamw(40, 40_000_000, "float32", 8), name="adamw_40m_8bit"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _even(d):
    """The multiple of 32, or of 160 for wide rows, at or below d."""
    step = 32 if d < 1024 else 160
    return max(32, d // step * step)


def draw(rng):
    op = rng.choice(["norm", "adapt", "adapt", "adamw"])
    dtype = rng.choice(list(TYPES))
    if op == "norm":
        dim = _spread(rng, 16, 8192)
        dim = _even(dim) if rng.random() < 0.6 else dim | 1
        return _norm(rng.choice(["forward", "gradient"]), _spread(rng, 1, min(65536, 64_000_000 // dim)), dim, dtype,
                     rng.choice([1, 1, 1, 4]))
    if op == "adapt":
        d_in, d_out = _spread(rng, 32, 4096), _spread(rng, 32, 4096)
        d_in, d_out = (_even(d_in), _even(d_out)) if rng.random() < 0.7 else (d_in | 1, d_out | 1)
        single = rng.random() < 0.25
        # (what a row costs in single precision is more than in 16 bits)
        most = int((60e9 if dtype == "float32" else 240e9) / (2 * d_in * d_out))
        rows = _spread(rng, 1, 128) if single else _spread(rng, 1, max(1, min(65536, most)))
        return _adapt("forward" if single else rng.choice(["forward", "gradient"]), rows, d_in, d_out, rng.choice([1, 3, 4, 8, 16, 24, 32, 64]),
                      _spread(rng, 1, 64), dtype, single)
    masters = dtype != "float32" and rng.random() < 0.7
    return _adamw(_spread(rng, 1, 60), _spread(rng, 2000, 60_000_000), dtype, rng.choice([32, 8]), masters, rng.random() < 0.3)


# ---- inputs

def _sizes(case):
    """Sizes of the tensors: most of the numbers in a few of them, odd ones, single numbers among the small ones."""
    rng = random.Random(case["tensors"] * 1_000_003 + case["numel"])
    weight = [math.exp(rng.uniform(0.0, 6.0)) for _ in range(case["tensors"])]
    total = sum(weight)
    return [max(1, int(case["numel"] * w / total)) for w in weight]


def _rows_of_requests(case, rng, device):
    """The adapter of every row.  Requests are runs of rows in the order they came in, one in eight without an adapter; or
    single rows, each a request of its own."""
    rows, adapters = case["rows"], case["adapters"]
    if case["single"]:
        # (different adapters while there are enough)
        order = [a for _ in range(-(-rows // adapters)) for a in rng.sample(range(adapters), adapters)][:rows]
        return torch.tensor(order, dtype=torch.int32, device=device)
    requests = max(1, min(rows, 2 * adapters + rng.randrange(adapters + 1)))
    ends = torch.tensor(sorted(rng.randrange(1, rows + 1) for _ in range(requests - 1)) + [rows], device=device)
    which = torch.tensor([-1 if rng.random() < 0.125 else rng.randrange(adapters) for _ in range(requests)], dtype=torch.int32, device=device)
    return which[torch.searchsorted(ends, torch.arange(rows, device=device), right=True)]


def prepare(case, seed):
    device = torch.device("cuda:0")
    gen = torch.Generator(device=device).manual_seed(seed)
    rng = random.Random(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dtype):
        return torch.randn(*shape, generator=gen, device=device, dtype=torch.float32).mul_(scale).to(dtype)

    if case["op"] == "norm":
        rows, dim, pitch = case["rows"], case["dim"], case["pitch"]
        # (rows of a wider array, as the scalars of features with higher orders are)
        x = torch.add(normal(rows, pitch * dim, scale=1.5), 0.3)[:, :dim]
        state = {"case": case, "x": x, "weight": torch.add(normal(dim, scale=0.2), 1.0), "bias": normal(dim, scale=0.1)}
        if case["direction"] == "gradient":
            wide = x.float()
            mean = wide.mean(1)
            state.update(dy=normal(rows, dim), mean=mean, rstd=torch.rsqrt((wide - mean[:, None]).square().mean(1) + EPS))
        return state
    if case["op"] == "adapt":
        rows, d_in, d_out, rank, n = case["rows"], case["d_in"], case["d_out"], case["rank"], case["adapters"]
        state = {"case": case, "x": normal(rows, d_in), "weight": normal(d_out, d_in, scale=d_in ** -0.5),
                 "A": normal(n, rank, d_in, scale=d_in ** -0.5), "B": normal(n, d_out, rank, scale=0.5 * rank ** -0.5),
                 "scale": torch.rand(n, generator=gen, device=device) + 0.5, "index": _rows_of_requests(case, rng, device)}
        if case["direction"] == "gradient":
            state["dy"] = normal(rows, d_out)
        return state

    # Parameters and moments lie in one array each, a tensor starting at a multiple of 256 numbers, or, packed, right behind the
    # one before it where a scale does not need that.
    sizes = _sizes(case)
    bits, masters = case["bits"], case["masters"]
    pad = 1 if case["packed"] and bits == 32 else BLOCK
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += -(-n // pad) * pad
    live = torch.zeros(at, dtype=torch.bool, device=device)
    for b, n in zip(starts, sizes):
        live[b:b + n] = True
    flat = lambda v: v.mul_(live)          # noqa: E731  (nothing between the tensors)
    value = flat(normal(at, scale=0.05, dtype=torch.float32))
    grad = flat(normal(at, scale=1e-3))
    state = {"case": case, "step": FIRST_STEP, "param": value.to(dtype), "master": value.to(dtype).float() if masters else None, "grad": grad}
    # moments after a few steps: between gradients much smaller and much larger than this one
    size = torch.exp(normal(at, scale=1.5, dtype=torch.float32)).mul_(live)
    m = normal(at, scale=3e-4, dtype=torch.float32).mul_(size)
    v = size.square_().mul_(1e-6).mul_(1 - BETA2 ** FIRST_STEP)
    if bits == 32:
        state.update(exp_avg=m, exp_avg_sq=v)
        state["moments"] = [(m[b:b + n], v[b:b + n]) for b, n in zip(starts, sizes)]
    else:
        sm, sv = m.view(-1, BLOCK).abs().amax(1), v.view(-1, BLOCK).amax(1)
        over = lambda a, s: torch.nan_to_num(a.view(-1, BLOCK) / s[:, None]).view(-1)          # noqa: E731
        cm = (torch.sqrt(over(m.abs(), sm)) * 127).round_().mul_(torch.sign(m)).to(torch.int8)
        cv = (torch.sqrt(torch.sqrt(over(v, sv))) * 255).round_().to(torch.uint8)
        cv = torch.where((v > 0) & (cv == 0), torch.ones_like(cv), cv)
        state.update(code_m=cm, scale_m=sm, code_v=cv, scale_v=sv)
        state["moments"] = [(cm[b:b + n], sm[b // BLOCK:(b + n + BLOCK - 1) // BLOCK], cv[b:b + n], sv[b // BLOCK:(b + n + BLOCK - 1) // BLOCK])
                            for b, n in zip(starts, sizes)]
        # the number of a value inside its tensor, which says where its rounding stands
        inside = torch.arange(at, device=device, dtype=torch.int32)
        for b, n in zip(starts, sizes):
            inside[b:b + -(-n // BLOCK) * BLOCK] -= b
        state["inside"] = inside
    state["params"] = [state["param"][b:b + n] for b, n in zip(starts, sizes)]
    state["grads"] = [grad[b:b + n] for b, n in zip(starts, sizes)]
    state["masters"] = [state["master"][b:b + n] for b, n in zip(starts, sizes)] if masters else None
    state["optimizer"] = None
    return state


# ---- the plain forms

def _plain_norm(s):
    x, w = s["x"].float(), s["weight"].float()
    if s["case"]["direction"] == "forward":
        mean = x.mean(1)
        centered = x - mean[:, None]
        rstd = torch.rsqrt(centered.square().mean(1) + EPS)
        y = centered * rstd[:, None] * w + s["bias"].float()
        return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}
    dy = s["dy"].float()
    hat = (x - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy * w
    dx = (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True)) * s["rstd"][:, None]
    return {"dx": dx.to(s["x"].dtype), "dweight": (dy * hat).sum(0).to(s["weight"].dtype), "dbias": dy.sum(0).to(s["bias"].dtype)}


def _plain_adapt(s):
    case, dtype = s["case"], s["x"].dtype
    n, rank, rows = case["adapters"], case["rank"], case["rows"]
    x, w, a, b = s["x"].float(), s["weight"].float(), s["A"].float(), s["B"].float()
    index, scale = s["index"].long(), s["scale"]
    if case["direction"] == "forward" and rows <= n:          # the adapters of few rows, taken out
        at = index.clamp(min=0)
        h = (a[at] * x[:, None, :]).sum(2) * torch.where(index >= 0, scale[at], torch.zeros_like(scale[at]))[:, None]
        return {"y": (x @ w.t() + (b[at] * h[:, None, :]).sum(2)).to(dtype)}
    # all adapters side by side; a row keeps what its own says
    mine = (index[:, None] == torch.arange(n, device=index.device)) * scale
    a_all = a.reshape(n * rank, -1)
    b_all = b.transpose(1, 2).reshape(n * rank, -1)
    h = ((x @ a_all.t()).view(rows, n, rank) * mine[:, :, None]).view(rows, n * rank)
    if case["direction"] == "forward":
        return {"y": (x @ w.t() + h @ b_all).to(dtype)}
    dy = s["dy"].float()
    g = ((dy @ b_all.t()).view(rows, n, rank) * mine[:, :, None]).view(rows, n * rank)
    return {"dx": (dy @ w + g @ a_all).to(dtype), "dA": (g.t() @ x).view(n, rank, -1).to(dtype),
            "dB": (h.t() @ dy).view(n, rank, -1).transpose(1, 2).contiguous().to(dtype)}


def _turn(inside, step, which):
    """Where the rounding of a moment stands at this step, in [0, 1): it moves on by steps that fill the interval evenly, so that
    what is rounded away at one step is made up for at others."""
    offset = ((2 * step + which) * 0x85EBCA6B + 2 ** 31) % 2 ** 32 - 2 ** 31
    return (((inside * (0x9E3779B1 - 2 ** 32) + offset) >> 8) & 0xFFFFFF).float() * 2.0 ** -24          # (32-bit numbers, modulo 2^32)


def _plain_adamw(s):
    case, t = s["case"], s["step"]
    s["step"] = t + 1
    p = s["master"] if case["masters"] else s["param"].float()
    g = s["grad"].float()
    if case["bits"] == 32:
        m, v = s["exp_avg"], s["exp_avg_sq"]
    else:
        m, v = _moments(s)
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g * (1 - BETA2) * g
    p = p * (1 - LR * DECAY) - (m * (LR / (1 - BETA1 ** t))) / (torch.sqrt(v) * (1 / math.sqrt(1 - BETA2 ** t)) + ADAM_EPS)
    if case["masters"]:
        s["master"].copy_(p)
    s["param"].copy_(p)
    if case["bits"] == 32:
        s["exp_avg"].copy_(m)
        s["exp_avg_sq"].copy_(v)
        return _adamw_out(s, m=s["exp_avg"], v=s["exp_avg_sq"])
    sm, sv = m.view(-1, BLOCK).abs().amax(1), v.view(-1, BLOCK).amax(1)
    by = lambda a, r: (a.view(-1, BLOCK) / torch.where(r > 0, r, torch.ones_like(r))[:, None]).view(-1)          # noqa: E731
    cm = torch.floor(torch.sqrt(by(m.abs(), sm)) * 127 + _turn(s["inside"], t, 0)).clamp_(max=127)
    cv = torch.floor(torch.sqrt(torch.sqrt(by(v, sv))) * 255 + _turn(s["inside"], t, 1)).clamp_(max=255)
    s["code_m"].copy_(torch.where(m < 0, -cm, cm))
    s["code_v"].copy_(torch.where(v > 0, cv.clamp(min=1), torch.zeros_like(cv)))
    s["scale_m"].copy_(sm)
    s["scale_v"].copy_(sv)
    m, v = _moments(s)
    return _adamw_out(s, m=m, v=v)


def _moments(s):
    """The moments that codes and scales stand for: scale c |c| / 127^2 and scale (c / 255)^4."""
    c = s["code_m"].float() * (1 / 127)
    d = s["code_v"].float() * (1 / 255)
    d = d * d
    return ((c * c.abs()).view(-1, BLOCK) * s["scale_m"][:, None]).view(-1), ((d * d).view(-1, BLOCK) * s["scale_v"][:, None]).view(-1)


def _adamw_out(s, m, v):
    out = {"param": s["param"], "exp_avg": m, "exp_avg_sq": v}
    if s["case"]["masters"]:
        out["master"] = s["master"]
    return out


# ---- the framework's operators

def _own(s):
    from symmetrix_amd import finetune
    case = s["case"]
    if case["op"] == "norm":
        if case["direction"] == "forward":
            y, mean, rstd = finetune.layer_norm_forward(s["x"], s["weight"], s["bias"], EPS)
            return {"y": y, "mean": mean, "rstd": rstd}
        dx, dw, db = finetune.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"])
        return {"dx": dx, "dweight": dw, "dbias": db}
    if case["op"] == "adapt":
        if case["direction"] == "forward":
            return {"y": finetune.adapted_linear_forward(s["x"], s["weight"], s["A"], s["B"], s["scale"], s["index"])}
        dx, da, db = finetune.adapted_linear_backward(s["dy"], s["x"], s["weight"], s["A"], s["B"], s["scale"], s["index"])
        return {"dx": dx, "dA": da, "dB": db}
    if s["optimizer"] is None:          # as a program makes its optimizer before the first step
        s["optimizer"] = finetune.AdamW(s["params"], lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY, state_bits=case["bits"],
                                        masters=s["masters"], states=s["moments"], step=FIRST_STEP - 1)
    s["optimizer"].step(s["grads"])
    if case["bits"] == 32:
        return _adamw_out(s, m=s["exp_avg"], v=s["exp_avg_sq"])
    m, v = finetune.moment_values(s["code_m"], s["scale_m"], s["code_v"], s["scale_v"])
    return _adamw_out(s, m=m, v=v)


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"norm": _plain_norm, "adapt": _plain_adapt, "adamw": _plain_adamw}[state["case"]["op"]](state)


# ---- what a pass cannot do without

def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "norm":
        cells, rows, dim = case["rows"] * case["dim"], case["rows"], case["dim"]
        if case["direction"] == "forward":
            return {"bytes": 2 * size * cells + 8 * rows + 2 * size * dim, "flops": 8 * cells}
        return {"bytes": 3 * size * cells + 8 * rows + 3 * size * dim, "flops": 14 * cells}
    if case["op"] == "adapt":
        rows, d_in, d_out, rank, n = case["rows"], case["d_in"], case["d_out"], case["rank"], case["adapters"]
        used = min(n, rows) * rank * (d_in + d_out)
        if case["direction"] == "forward":
            return {"bytes": size * (rows * (d_in + d_out) + d_in * d_out + used) + 4 * rows,
                    "flops": 2 * rows * (d_in * d_out + rank * (d_in + d_out))}
        return {"bytes": size * (rows * (2 * d_in + d_out) + d_in * d_out + used + n * rank * (d_in + d_out)) + 4 * rows,
                "flops": 2 * rows * (d_in * d_out + 3 * rank * (d_in + d_out))}
    numel = sum(_sizes(case))
    bytes_each = size + (size + 8 if case["masters"] else 2 * size) + (16 if case["bits"] == 32 else 4 + 16 / BLOCK)
    if case["bits"] == 8:
        bytes_each += 8 + 2 + 8 / BLOCK          # the moments as the numbers they stand for
    return {"bytes": numel * bytes_each, "flops": 16 * numel}


# ---- in 64 bits, from the definitions

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x, w = s["x"].double(), s["weight"].double()
        if case["direction"] == "forward":
            var, mean = torch.var_mean(x, 1, correction=0)
            rstd = 1.0 / torch.sqrt(var + EPS)
            return {"y": (x - mean[:, None]) * (rstd[:, None] * w) + s["bias"].double(), "mean": mean, "rstd": rstd}
        mean, rstd, dy = s["mean"].double()[:, None], s["rstd"].double()[:, None], s["dy"].double()
        hat = rstd * (x - mean)
        inner = (dy * w * hat).sum(1, keepdim=True) / case["dim"]
        outer = (dy * w).sum(1, keepdim=True) / case["dim"]
        return {"dx": rstd * (dy * w - (outer + hat * inner)), "dweight": torch.einsum("ij,ij->j", dy, hat), "dbias": dy.sum(0)}
    if case["op"] == "adapt":
        x, w, index = s["x"].double(), s["weight"].double(), s["index"].tolist()
        rows_of = {}
        for i, a in enumerate(index):
            rows_of.setdefault(a, []).append(i)
        forward = case["direction"] == "forward"
        if forward:
            out = {"y": torch.matmul(x, w.t())}
        else:
            dy = s["dy"].double()
            out = {"dx": torch.matmul(dy, w), "dA": torch.zeros_like(s["A"], dtype=torch.float64), "dB": torch.zeros_like(s["B"], dtype=torch.float64)}
        for k, rows in rows_of.items():
            if k < 0:
                continue
            at = torch.tensor(rows, device=x.device)
            A, B, c = s["A"][k].double(), s["B"][k].double(), float(s["scale"][k])
            if forward:
                out["y"][at] += c * torch.matmul(torch.matmul(x[at], A.t()), B.t())
            else:
                up = c * torch.matmul(dy[at], B)
                out["dx"][at] += torch.matmul(up, A)
                out["dA"][k] = torch.matmul(up.t().contiguous(), x[at])
                out["dB"][k] = torch.matmul(dy[at].t().contiguous(), c * torch.matmul(x[at], A.t()))
        return out
    t = s["step"]
    p = (s["master"] if case["masters"] else s["param"]).double()
    g = s["grad"].double()
    if case["bits"] == 32:
        m, v = s["exp_avg"].double(), s["exp_avg_sq"].double()
    else:
        wide = lambda c, r: c * r.double().repeat_interleave(BLOCK)          # noqa: E731
        m = wide(torch.sign(s["code_m"].double()) * (s["code_m"].double() / 127) ** 2, s["scale_m"])
        v = wide((s["code_v"].double() / 255) ** 4, s["scale_v"])
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    p = p - LR * DECAY * p - LR * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + ADAM_EPS)
    out = {"param": p, "exp_avg": m, "exp_avg_sq": v} if case["bits"] == 32 else {"param": p, "exp_avg": None, "exp_avg_sq": None}
    if case["masters"]:
        out["master"] = p
    return out
