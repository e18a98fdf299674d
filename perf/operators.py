"""Feed-forwards with weights in microscaled 4-bit numbers (MXFP4): what is computed, in cases that can be timed and checked.

Four operators:

  quantize   a matrix or a stack of matrices into blocks of 32 four-bit numbers with a power of two each, and back to the values
             they stand for: what loading a model does once
  linear     x W^T (+ bias): a feed-forward's last product, or an ungated one's first
  gated      act(x G^T) * (x U^T): a gated feed-forward's first half
  experts    a whole layer of routed experts for the rows of a step, from their chosen experts and weights to its output

The format is the Open Compute Project's MXFP4: 32 consecutive values of a row share 2^s, s = floor(log2(largest)) - 2 within
-127 .. 127, and each is the nearest (ties to even) of 0, 1/2, 1, 3/2, 2, 3, 4, 6 times it, with a sign, the largest of them beyond 6.
Activations are bfloat16, sums 32-bit.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
BLOCK = 32


def listed():
    return [
        # a small odd matrix of a checkpoint in 32 bits: rows that end inside a block
        {"name": "quantize 520 x 1000 f32", "op": "quantize", "groups": 1, "n": 520, "k": 1000, "dtype": "float32"},
        # the gate and up matrices of a layer of 32 experts, as loading an 8B model meets them 22 times
        {"name": "quantize 32 experts", "op": "quantize", "groups": 64, "n": 1792, "k": 2048, "dtype": "bfloat16"},
        # the down product of one decode row
        {"name": "linear 1 x 2048 x 7168", "op": "linear", "m": 1, "n": 2048, "k": 7168, "bias": False, "out": "float32"},
        # ... of a step of some requests, with a bias, sizes that fit no tile
        {"name": "linear 37 x 1000 x 2731", "op": "linear", "m": 37, "n": 1000, "k": 2731, "bias": True, "out": "bfloat16"},
        # ... of a prompt
        {"name": "linear 2048 x 2048 x 7168", "op": "linear", "m": 2048, "n": 2048, "k": 7168, "bias": False, "out": "float32"},
        # the first half of a dense layer: a decode step of 8 requests
        {"name": "gated 8 x 7168 x 2048", "op": "gated", "m": 8, "n": 7168, "k": 2048, "act": "silu"},
        # a short prompt, sizes that fit no tile
        {"name": "gated 150 x 2500 x 1096", "op": "gated", "m": 150, "n": 2500, "k": 1096, "act": "gelu"},
        # a long prompt's portion
        {"name": "gated 2048 x 7168 x 2048", "op": "gated", "m": 2048, "n": 7168, "k": 2048, "act": "silu"},
        # an expert layer of the 8B model: one decode row
        {"name": "experts 1 row", "op": "experts", "m": 1, "e": 32, "top": 4, "n": 1792, "k": 2048, "act": "silu", "form": "gated"},
        # ... a step of 8 requests
        {"name": "experts 8 rows", "op": "experts", "m": 8, "e": 32, "top": 4, "n": 1792, "k": 2048, "act": "silu", "form": "gated"},
        # many small experts and a step of some dozen requests
        {"name": "experts 45 rows of 64", "op": "experts", "m": 45, "e": 64, "top": 6, "n": 768, "k": 2048, "act": "silu", "form": "gated"},
        # ... a long prompt's portion
        {"name": "experts 2048 rows", "op": "experts", "m": 2048, "e": 32, "top": 4, "n": 1792, "k": 2048, "act": "silu", "form": "gated"},
    ]


def draw(rng):
    def log(low, high):
        return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))

    op = rng.choice(("quantize", "linear", "gated", "experts"))
    while True:
        if op == "quantize":
            case = {"op": op, "groups": log(1, 64), "n": log(1, 8192), "k": log(1, 8192), "dtype": rng.choice(list(DTYPES))}
            if case["groups"] * case["n"] * case["k"] > 64 * 1792 * 2048 // (2 if case["dtype"] == "float32" else 1):
                continue
        elif op == "linear":
            case = {"op": op, "m": log(1, 4096), "n": log(8, 8192), "k": log(16, 8192), "bias": rng.random() < 0.5,
                    "out": rng.choice(list(DTYPES))}
            if case["m"] * case["n"] * case["k"] > 2048 * 2048 * 7168:
                continue
        elif op == "gated":
            case = {"op": op, "m": log(1, 4096), "n": log(8, 7168), "k": log(16, 4096), "act": rng.choice(("silu", "gelu", "relu2"))}
            if case["m"] * case["n"] * case["k"] > 2048 * 2048 * 7168:
                continue
        else:
            e = log(2, 64)
            case = {"op": op, "m": log(1, 2048), "e": e, "top": rng.randint(1, min(8, e)), "n": log(16, 2048), "k": log(32, 2560),
                    "act": rng.choice(("silu", "gelu", "relu2")), "form": rng.choice(("gated", "gated", "ungated", "weighed input"))}
            if case["m"] * case["top"] * case["n"] * case["k"] > 2048 * 4 * 1792 * 2048 or e * case["n"] * case["k"] > 32 * 1792 * 2048:
                continue
        return case


# ---- inputs ----

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _matrix(g, groups, n, k, dtype):
    """Weights as trained ones are spread: rows of different size, a few columns that stand out."""
    w = torch.randn(groups, n, k, generator=g, device=DEVICE, dtype=dtype) * 0.02
    w *= torch.exp(0.5 * torch.randn(groups, n, 1, generator=g, device=DEVICE)).to(dtype)
    w *= torch.exp(0.3 * torch.randn(1, 1, k, generator=g, device=DEVICE)).to(dtype)
    return w


def _rows(g, m, k):
    """Normed rows with a few channels that stand out."""
    x = torch.randn(m, k, generator=g, device=DEVICE) * torch.exp(0.5 * torch.randn(k, generator=g, device=DEVICE))
    return x.to(torch.bfloat16)


def _inputs(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op == "quantize":
        w = _matrix(g, case["groups"], case["n"], case["k"], DTYPES[case["dtype"]])
        w[:, : case["n"] // 16 + 1, : case["k"] // 2] = 0      # pruned pieces: blocks of zeros
        return {"w": w}
    x = _rows(g, case["m"], case["k"])
    if op == "linear":
        bias = torch.randn(case["n"], generator=g, device=DEVICE) if case["bias"] else None
        return {"x": x, "w": _matrix(g, 1, case["n"], case["k"], torch.bfloat16), "bias": bias}
    if op == "gated":
        return {"x": x, "w": _matrix(g, 2, case["n"], case["k"], torch.bfloat16)}
    e, gates = case["e"], 1 if case["form"] == "ungated" else 2
    scores = torch.randn(case["m"], e, generator=g, device=DEVICE) + 0.4 * torch.randn(e, generator=g, device=DEVICE)
    wts, ids = torch.sigmoid(scores).topk(case["top"], dim=1)
    return {"x": x, "ids": ids.to(torch.int32).contiguous(), "wts": (wts / wts.sum(1, keepdim=True)).contiguous(),
            "w": _matrix(g, gates * e, case["n"], case["k"], torch.bfloat16), "down": _matrix(g, e, case["k"], case["n"], torch.bfloat16)}


# ---- the plain form ----

def _power(s):
    """2^s in 64 bits from whole s in -1022 .. 1023, exactly."""
    return ((s.to(torch.int64) + 1023) << 52).view(torch.float64)


def _encode(w):
    """(elements in halves as whole numbers -12 .. 12 [.., blocks, 32], exponents [.., blocks, 1])."""
    k = w.shape[-1]
    v = torch.nn.functional.pad(w, (0, -k % BLOCK)).unflatten(-1, (-1, BLOCK)).float()
    s = (torch.frexp(v.abs().amax(-1, keepdim=True))[1] - 3).clamp(-127, 127)
    s = torch.where((v == 0).all(-1, keepdim=True), -127, s)
    y = v * _power(-s)
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
    y = (torch.round(y / step) * step).clamp(-6, 6)
    return (2 * y).to(torch.int8), s.to(torch.int16)


def _values(q, k):
    """The values in 32 bits of what `_encode` gave."""
    halves, s = q
    return (halves * _power(s - 1)).float().flatten(-2)[..., :k]


def _activation(z, act):
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2.0)))
    return torch.square(torch.clamp(z, min=0))


def _chosen(state):
    """Rows of one expert side by side: (the experts chosen at all, each pair's expert among them and its place there, the most rows)."""
    ids = state["ids"].long().flatten()
    experts, which = torch.unique(ids, return_inverse=True)
    order = torch.argsort(which, stable=True)
    counts = torch.bincount(which)
    place = torch.empty_like(which)
    place[order] = torch.arange(len(ids), device=ids.device) - (torch.cumsum(counts, 0) - counts)[which[order]]
    return experts, which, place, int(counts.max())


def _plain(case, state):
    op = case["op"]
    if op == "quantize":
        w = state["w"]
        return _values(_encode(w), w.shape[-1]).to(w.dtype)
    x, k = state["x"].float(), case["k"]
    if op == "linear":
        c = x @ _values(state["w"], k)[0].T
        return (c if state["bias"] is None else c + state["bias"]).to(DTYPES[case["out"]])
    if op == "gated":
        w = _values(state["w"], k)
        return (_activation(x @ w[0].T, case["act"]) * (x @ w[1].T)).to(torch.bfloat16)
    m, top, n = case["m"], case["top"], case["n"]
    experts, which, place, most = _chosen(state)
    rows = x.repeat_interleave(top, 0)
    wts = state["wts"].flatten()[:, None]
    xs = x.new_zeros(len(experts), most, k)
    xs[which, place] = rows * wts if case["form"] == "weighed input" else rows
    halves, s = state["w"]
    w = _values((halves.unflatten(0, (case["e"], -1))[experts], s.unflatten(0, (case["e"], -1))[experts]), k)
    up = xs @ w[:, -1].transpose(1, 2)
    a = _activation(up, case["act"]) if case["form"] == "ungated" else _activation(xs @ w[:, 0].transpose(1, 2), case["act"]) * up
    y = (a @ _values(tuple(t[experts] for t in state["down"]), n).transpose(1, 2))[which, place]
    y = y if case["form"] == "weighed input" else y * wts
    return y.unflatten(0, (m, top)).sum(1).to(torch.bfloat16)


# ---- what the tools call ----

def prepare(case, seed):
    """Rows as they come, weights as a program keeps them: quantised once."""
    state = _inputs(case, seed)
    if case["op"] == "quantize":
        return {"case": case, **state}
    if own:
        from tandemllm_b200.kernels import mxfp4, tensorcore
        from tandemllm_b200.parts.base import Runtime
        state["runtime"] = Runtime(torch.device(DEVICE), torch.bfloat16)
        tensorcore.enable(state["runtime"])
        if case["op"] == "linear":
            state["w"] = mxfp4.quantize(state["w"][0])
        else:
            state["w"] = mxfp4.quantize(state["w"])
        if case["op"] == "experts":
            state["down"] = mxfp4.quantize(state["down"])
    else:
        state["w"] = _encode(state["w"])
        if case["op"] == "experts":
            state["down"] = _encode(state["down"])
    return {"case": case, **state}


def run(state):
    case = state["case"]
    if not own:
        return _plain(case, state)
    from tandemllm_b200.kernels import mxfp4
    op = case["op"]
    if op == "quantize":
        return mxfp4.quantize(state["w"]).values(state["w"].dtype)
    if op == "linear":
        return mxfp4.linear(state["runtime"], state["x"], state["w"], state["bias"], out_dtype=DTYPES[case["out"]])
    if op == "gated":
        return mxfp4.gated(state["runtime"], state["x"], state["w"], case["act"])
    return mxfp4.experts(state["runtime"], state["x"], state["ids"], state["wts"], state["w"], state["down"], case["act"],
                         weigh="input" if case["form"] == "weighed input" else "output")


def work(case):
    n, k = case["n"], case["k"]
    packed = lambda count: count * 17 / 32      # noqa: E731
    if case["op"] == "quantize":
        count = case["groups"] * n * k
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": 2 * size * count + packed(count), "flops": 4 * count}
    m = case["m"]
    if case["op"] == "linear":
        return {"bytes": 2 * m * k + packed(n * k) + (4 if case["out"] == "float32" else 2) * m * n, "flops": 2 * m * n * k}
    if case["op"] == "gated":
        return {"bytes": 2 * m * k + packed(2 * n * k) + 2 * m * n, "flops": 4 * m * n * k}
    e, top, matrices = case["e"], case["top"], 2 if case["form"] == "ungated" else 3
    read = e * (1 - (1 - top / e) ** m)         # experts that some row chooses, all as likely
    return {"bytes": 4 * m * k + 8 * m * top + packed(read * matrices * n * k), "flops": 2 * m * top * matrices * n * k}


# ---- the definition in 64 bits ----

def _rounded64(w):
    """Each value by the format's definition: the levels of its block, the nearest of them, the even one of two."""
    k = w.shape[-1]
    levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=w.device)
    between = (levels[1:] + levels[:-1]) / 2
    out = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
    for first in range(0, k, BLOCK):
        v = w[..., first : first + BLOCK].double()
        top = v.abs().amax(-1, keepdim=True)
        _, e = torch.frexp(top)
        scale = torch.where(top > 0, torch.ldexp(torch.ones_like(top), (e - 3).clamp(-127, 127)), torch.ones_like(top))
        y = v.abs() / scale
        low, high = torch.searchsorted(between, y, right=False), torch.searchsorted(between, y, right=True)
        at = torch.where(low == high, low, torch.where(low % 2 == 0, low, high))      # on a border: the even code
        out[..., first : first + BLOCK] = torch.sign(v) * levels[at] * scale
    return out


def exact(case, seed):
    state = _inputs(case, seed)
    if case["op"] == "quantize":
        w = state["w"]
        return torch.stack([_rounded64(one) for one in w]).to(w.dtype)
    x = state["x"].double()
    act = {"silu": lambda z: z * torch.sigmoid(z), "gelu": lambda z: torch.nn.functional.gelu(z), "relu2": lambda z: torch.relu(z) ** 2}
    if case["op"] == "linear":
        c = torch.nn.functional.linear(x, _rounded64(state["w"][0]))
        return c if state["bias"] is None else c + state["bias"].double()
    if case["op"] == "gated":
        return act[case["act"]](torch.nn.functional.linear(x, _rounded64(state["w"][0]))) * torch.nn.functional.linear(x, _rounded64(state["w"][1]))
    f = act[case["act"]]
    out = torch.zeros_like(x)
    for e in range(case["e"]):
        rows, slots = torch.nonzero(state["ids"] == e, as_tuple=True)
        if not len(rows):
            continue
        weight, xe = state["wts"][rows, slots].double()[:, None], x[rows]
        if case["form"] == "weighed input":
            xe, weight = xe * weight, torch.ones_like(weight)
        if case["form"] == "ungated":
            a = f(torch.nn.functional.linear(xe, _rounded64(state["w"][e])))
        else:
            a = f(torch.nn.functional.linear(xe, _rounded64(state["w"][2 * e]))) * torch.nn.functional.linear(xe, _rounded64(state["w"][2 * e + 1]))
        out.index_add_(0, rows, weight * torch.nn.functional.linear(a, _rounded64(state["down"][e])))
    return out
