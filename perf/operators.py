"""Cases of the training operators: the latent-code lookup and its gradient, the dense 16-bit layer with bias, activation and
residual in its epilogue, and the global gradient norm with clipping.

``own`` False: plain torch in 32 bits (64 for long sums); True: the framework's operators (nphm_amd.train_ops)."""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
ACTIVATIONS = ("none", "relu", "silu", "gelu", "softplus")

# parameter shapes of the identity decoder (39 anchors: 24 weight sets of five ensemble layers, and the anchor head)
DECODER = ((24, 200, 99), (24, 200), (24, 101, 200), (24, 101), (24, 200, 200), (24, 200), (24, 200, 200), (24, 200),
           (24, 1, 200), (24, 1), (256, 64), (256,), (256, 256), (256,), (117, 256), (117,))


def listed():
    return [
        # the codes of one batch of subjects, forward and gradient: latency counts
        {"name": "codes batch", "op": "lookup", "way": "both", "dtype": "fp32", "rows": 24, "dim": 1344, "count": 16, "scale": 1.0,
         "padding": -1, "skewed": False},
        # rows of a large table for a long packed batch
        {"name": "token rows", "op": "lookup", "way": "forward", "dtype": "bf16", "rows": 50000, "dim": 4096, "count": 16384, "scale": 64.0,
         "padding": -1, "skewed": False},
        # gradient of a large table: few rows take most of the batch, one of them is padding
        {"name": "token gradient", "op": "lookup", "way": "gradient", "dtype": "bf16", "rows": 50000, "dim": 2048, "count": 32768,
         "scale": 1.0, "padding": 3, "skewed": True},
        # odd table, odd width: rows that no wide load fits
        {"name": "odd gradient", "op": "lookup", "way": "gradient", "dtype": "fp16", "rows": 10007, "dim": 1001, "count": 4097, "scale": 0.5,
         "padding": -1, "skewed": True},
        # the identity decoder's sixteen gradients, as its trainer clips them
        {"name": "clip decoder", "op": "clip", "dtype": "fp32", "tensors": 0, "mean": 0, "sizes": 0, "packed": False, "limit": 0.1},
        # a large model's gradients
        {"name": "clip large", "op": "clip", "dtype": "bf16", "tensors": 290, "mean": 1 << 20, "sizes": 5, "packed": False, "limit": 1.0},
        # many small ragged tensors, one behind the other in a bucket: no start is aligned
        {"name": "clip ragged", "op": "clip", "dtype": "fp16", "tensors": 500, "mean": 3000, "sizes": 9, "packed": True, "limit": 1e9},
        # few rows through a layer: the weight is what has to be read
        {"name": "layer few rows", "op": "layer", "train": False, "dtype": "bf16", "m": 5, "k": 512, "n": 1024, "act": "silu", "bias": True,
         "residual": False},
        # the global network's hidden layer on a batch of points, forward and backward
        {"name": "layer hidden", "op": "layer", "train": True, "dtype": "bf16", "m": 16384, "k": 1024, "n": 1024, "act": "softplus",
         "bias": True, "residual": False},
        # its first layer: 512 code entries and 3 coordinates, odd rows
        {"name": "layer odd", "op": "layer", "train": True, "dtype": "bf16", "m": 4095, "k": 515, "n": 1024, "act": "softplus", "bias": True,
         "residual": False},
        # a wide layer on a long batch, forward
        {"name": "layer wide", "op": "layer", "train": False, "dtype": "bf16", "m": 16384, "k": 4096, "n": 16384, "act": "gelu", "bias": True,
         "residual": False},
        # the product back to the residual stream, forward and backward
        {"name": "layer residual", "op": "layer", "train": True, "dtype": "fp16", "m": 8192, "k": 4096, "n": 4096, "act": "none",
         "bias": True, "residual": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("lookup", "clip", "layer"))
    if op == "lookup":
        rows = _log(rng, 8, 60000)
        return {"op": op, "way": rng.choice(("forward", "gradient", "both")), "dtype": rng.choice(sorted(DTYPES)), "rows": rows,
                "dim": _log(rng, 16, 4096), "count": _log(rng, 1, 40000), "scale": rng.choice((1.0, 0.5, 27.7)),
                "padding": rng.choice((-1, rng.randrange(rows))), "skewed": rng.random() < 0.5}
    if op == "clip":
        tensors = _log(rng, 1, 600)
        return {"op": op, "dtype": rng.choice(sorted(DTYPES)), "tensors": tensors, "mean": _log(rng, 8, (1 << 28) // tensors // 2),
                "sizes": rng.randrange(1000), "packed": rng.random() < 0.5, "limit": rng.choice((0.1, 1.0, 1e9))}
    m, k = _log(rng, 1, 16384), _log(rng, 8, 4096)
    return {"op": op, "train": rng.random() < 0.5, "dtype": rng.choice(("bf16", "fp16")), "m": m, "k": k,
            "n": _log(rng, 1, min(16384, (1 << 38) // (m * k))), "act": rng.choice(ACTIVATIONS), "bias": rng.random() < 0.7,
            "residual": rng.random() < 0.4}


def _sizes(case):
    """element counts of a clip case's tensors: the decoder's, or spread around a mean"""
    if not case["tensors"]:
        return [math.prod(s) for s in DECODER]
    r = random.Random(case["sizes"])
    return [max(1, int(case["mean"] * r.uniform(0.1, 1.9))) for _ in range(case["tensors"])]


def _views(flat, sizes, step):
    """consecutive views of `flat` that start at multiples of `step` elements"""
    at, got = 0, []
    for n in sizes:
        got.append(flat[at:at + n])
        at += -(-n // step) * step
    return got


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=gen).mul_(std).to(t)

    if case["op"] == "lookup":
        v, d, n = case["rows"], case["dim"], case["count"]
        u = torch.rand(n, device="cuda", generator=gen, dtype=torch.float64)
        idx = ((u * math.log(v)).exp() - 1 if case["skewed"] else u * v).long().clamp_(0, v - 1)
        state = {"case": case, "idx": idx}
        if case["way"] != "gradient":
            state["table"] = normal(v, d, std=0.1 / math.sqrt(d))
        if case["way"] != "forward":
            state["grad"] = normal(n, d)
        return state
    if case["op"] == "clip":
        sizes = _sizes(case)
        step = 1 if case["packed"] else 16
        total = sum(-(-n // step) * step for n in sizes)
        flat = normal(total, std=1e-3)
        out = torch.zeros(total, device="cuda", dtype=t)
        return {"case": case, "grads": _views(flat, sizes, step), "clipped": _views(out, sizes, step), "flat": out}
    m, k, n = case["m"], case["k"], case["n"]
    state = {"case": case, "x": normal(m, k), "weight": normal(n, k, std=1 / math.sqrt(k)),
             "bias": normal(n, std=0.1) if case["bias"] else None, "residual": normal(m, n) if case["residual"] else None}
    if case["train"]:
        state["grad"] = normal(m, n)
        for name in ("x", "weight", "bias", "residual"):
            if state[name] is not None:
                state[name].requires_grad_()
    return state


# ---- plain forms ------------------------------------------------------------------------------------------------------------

def _plain_lookup(table, idx, scale):
    return (table[idx].float() * scale).to(table.dtype)


def _plain_lookup_grad(grad, idx, rows, scale, padding):
    g = grad.float() * scale
    if padding >= 0:
        g = torch.where((idx == padding)[:, None], torch.zeros((), device=g.device), g)
    return torch.zeros(rows, grad.shape[1], device=g.device).index_add_(0, idx, g).to(grad.dtype)


def _plain_clip(grads, limit, out):
    norm = torch.stack([g.float().square().sum(dtype=torch.float64) for g in grads]).sum().sqrt()
    coef = (limit / (norm + 1e-6)).clamp(max=1.0).float()
    return norm.float(), [o.copy_(g.float() * coef) for g, o in zip(grads, out)]


def _beta(case):
    return 100.0 if case["act"] == "softplus" else 1.0


def _plain_act(z, act, beta):
    """(a(z), a'(z)); a' None for the identity"""
    if act == "none":
        return z, None
    if act == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    bz = z * beta
    return torch.where(bz > 20, z, torch.log1p(torch.exp(bz.clamp(max=20))) / beta), torch.sigmoid(bz)


def _plain_layer(s, case):
    t = s["x"].dtype
    with torch.no_grad():
        x, w = s["x"].float(), s["weight"].float()
        z = x @ w.t()
        if s["bias"] is not None:
            z = z + s["bias"].float()
        y, slope = _plain_act(z, case["act"], _beta(case))
        if s["residual"] is not None:
            y = y + s["residual"].float()
        if not case["train"]:
            return {"y": y.to(t)}
        gz = s["grad"].float() if slope is None else s["grad"].float() * slope
        got = {"y": y.to(t), "x": (gz @ w).to(t), "weight": (gz.t() @ x).to(t)}
        if s["bias"] is not None:
            got["bias"] = gz.sum(0).to(t)
        if s["residual"] is not None:
            got["residual"] = s["grad"].clone()
        return got


# ---- one pass ---------------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    if case["op"] == "lookup":
        got = {}
        if case["way"] != "gradient":
            got["rows"] = _plain_lookup(state["table"], state["idx"], case["scale"])
        if case["way"] != "forward":
            got["table"] = _plain_lookup_grad(state["grad"], state["idx"], case["rows"], case["scale"], case["padding"])
        return got
    if case["op"] == "clip":
        norm, _ = _plain_clip(state["grads"], case["limit"], state["clipped"])
        return {"norm": norm, "clipped": state["flat"]}
    return _plain_layer(state, case)


def _own(state, case):
    from nphm_amd import train_ops
    if case["op"] == "lookup":
        got, padding = {}, case["padding"] if case["padding"] >= 0 else None
        if case["way"] != "gradient":
            got["rows"] = train_ops.lookup_rows(state["table"], state["idx"], scale=case["scale"], padding_idx=padding)
        if case["way"] != "forward":
            got["table"] = train_ops.lookup_rows_grad(state["grad"], state["idx"], case["rows"], scale=case["scale"], padding_idx=padding)
        return got
    if case["op"] == "clip":
        norm, _ = train_ops.clip_grads(state["grads"], case["limit"], out=state["clipped"])
        return {"norm": norm, "clipped": state["flat"]}
    y = train_ops.linear_act(state["x"], state["weight"], state["bias"], activation=case["act"], beta=_beta(case), residual=state["residual"])
    if not case["train"]:
        return {"y": y}
    names = [n for n in ("x", "weight", "bias", "residual") if state[n] is not None]
    return {"y": y.detach(), **dict(zip(names, torch.autograd.grad(y, [state[n] for n in names], state["grad"])))}


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "lookup":
        v, d, n = case["rows"], case["dim"], case["count"]
        distinct = v * -math.expm1(n * math.log1p(-1 / v))
        moved = 0
        if case["way"] != "gradient":
            moved += (distinct + n) * d * e
        if case["way"] != "forward":
            moved += (n + v) * d * e
        return {"bytes": moved + 8 * n, "flops": 0}
    if case["op"] == "clip":
        n = sum(_sizes(case))
        return {"bytes": 2 * n * e, "flops": 3 * n}
    m, k, n = case["m"], case["k"], case["n"]
    moved = (m * k + n * k + m * n) * e + (n * e if case["bias"] else 0) + (m * n * e if case["residual"] else 0)
    if not case["train"]:
        return {"bytes": moved, "flops": 2 * m * n * k}
    return {"bytes": moved + (m * n + m * k + n * k) * e + (n * e if case["bias"] else 0), "flops": 6 * m * n * k}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "lookup":
        got = {}
        if case["way"] != "gradient":
            got["rows"] = torch.index_select(s["table"].double(), 0, s["idx"]) * case["scale"]
        if case["way"] != "forward":
            keep = s["idx"] != case["padding"]
            total = torch.zeros(case["rows"], case["dim"], device="cuda", dtype=torch.float64)
            total.index_put_((s["idx"][keep],), s["grad"][keep].double(), accumulate=True)
            got["table"] = total * case["scale"]
        return got
    if case["op"] == "clip":
        norm = math.sqrt(math.fsum(float(g.double().pow(2).sum()) for g in s["grads"]))
        factor = min(1.0, case["limit"] / (norm + 1e-6))
        flat = torch.zeros(s["flat"].shape, device="cuda", dtype=torch.float64)
        step = 1 if case["packed"] else 16
        for g, o in zip(s["grads"], _views(flat, _sizes(case), step)):
            o.copy_(g.double() * factor)
        return {"norm": norm, "clipped": flat}
    leaves = {n: s[n].detach().double().requires_grad_() for n in ("x", "weight", "bias", "residual") if s[n] is not None}
    z = torch.nn.functional.linear(leaves["x"], leaves["weight"], leaves.get("bias"))
    f = torch.nn.functional
    y = {"none": lambda v: v, "relu": f.relu, "silu": f.silu, "gelu": f.gelu,
         "softplus": lambda v: f.softplus(v, beta=_beta(case))}[case["act"]](z)
    if "residual" in leaves:
        y = y + leaves["residual"]
    if not case["train"]:
        return {"y": y.detach()}
    return {"y": y.detach(), **dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), s["grad"].double())))}
