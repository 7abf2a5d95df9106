"""The dense products of a mixed batch and their 8-bit forms: what is timed, on which sizes.

A graph batch is a block of rows per graph (``group_ptr``), and every graph belongs to one of several models
(``model_of_group``); a layer multiplies its rows with that model's weights, in floating point or in 8-bit integers
with a scale for each row and each output channel.  Four operators:

    quantize       rows of floats -> rows of int8 and one float32 scale per row
    int8           Y = act((Hq . Wq^T) * row scale * channel scale + bias)
    grouped        Y[rows of group g] = act(H . W[model of g]^T + bias[model of g])
    grouped_int8   the two together

``own`` selects between the elementary torch form and the framework's entry points.
"""
import random

import torch

own = False

LEAKY = 0.2
F32, BF16, F16 = "float32", "bfloat16", "float16"
SIZE = {F32: 4, BF16: 2, F16: 2}

_engine = None


def _eng():
    global _engine
    if _engine is None:
        from distgcn_amd.engine import Engine
        _engine = Engine("cuda:0")
    return _engine


# ---- the cases ------------------------------------------------------------------------------------------------------------------

def listed():
    def quantize(name, rows, cols, dtype, pad=0):
        return {"name": name, "op": "quantize", "rows": rows, "cin": cols, "dtype": dtype, "pad": pad}

    def int8(name, rows, cin, ctot, dtype, act, bias, pad=0):
        return {"name": name, "op": "int8", "rows": rows, "cin": cin, "ctot": ctot, "dtype": dtype, "act": act, "bias": bias, "pad": pad}

    def grouped(name, op, rows, cin, ctot, dtype, groups, models, split, act, bias, layout, pad=0):
        return {"name": name, "op": op, "rows": rows, "cin": cin, "ctot": ctot, "dtype": dtype, "groups": groups, "models": models,
                "split": split, "act": act, "bias": bias, "layout": layout, "pad": pad}

    return [
        # the hidden activations of 500 graphs of 200 vertices, 32 features each, before an 8-bit layer
        quantize("quantize-hidden", 100000, 32, F32),
        # a wide stack's activations in half precision, and the weights of such a layer when a model is loaded
        quantize("quantize-wide", 16384, 4096, BF16),
        # one row: what a single token's or a single vertex's product waits for
        quantize("quantize-one-row", 1, 4096, F16),
        # one layer of a 128-wide stack over the same 500 graphs: both supports' weights side by side, float32 for the aggregation
        int8("int8-wide-layer", 100000, 128, 256, F32, "linear", False),
        # a long prompt or a large batch through a large layer
        int8("int8-prompt", 8192, 4096, 4096, BF16, "relu", True),
        # a handful of tokens through the same layer: the weights' bytes are the cost
        int8("int8-tokens", 5, 4096, 4096, BF16, "linear", True),
        # the hidden layer of 500 graphs of 100 to 300 vertices, each under one of four checkpoints
        grouped("grouped-hidden", "grouped", 100000, 32, 64, F32, 500, 4, "graphs", "linear", False, 1),
        # the last layer of 4 000 such graphs under 46 checkpoints: one output for each of the two supports
        grouped("grouped-last", "grouped", 800000, 32, 2, F32, 4000, 46, "graphs", "linear", False, 2),
        # experts of a layer during a prompt, uneven loads
        grouped("grouped-experts", "grouped", 8192, 2048, 4096, BF16, 8, 8, "experts", "linear", False, 3),
        # the experts of a few tokens: most groups hold one row or none; an odd row stride
        grouped("grouped-tokens", "grouped", 24, 2048, 1024, F16, 64, 64, "experts", "leaky_relu", True, 4, pad=3),
        # many experts in 8 bits during a prompt, odd widths
        grouped("grouped-int8-experts", "grouped_int8", 16384, 2000, 2050, F16, 64, 64, "experts", "leaky_relu", True, 5),
        # and for a few tokens
        grouped("grouped-int8-tokens", "grouped_int8", 16, 2048, 2048, BF16, 64, 64, "experts", "linear", False, 6),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


MAX_FLOPS = 2 * 8192 * 4096 * 4096
MAX_BYTES = 200 * 1000 * 1000


def draw(rng):
    while True:
        op = rng.choice(["quantize", "int8", "grouped", "grouped_int8"])
        pad = rng.choice([0, 0, 0, 1, 5, 16, 32])
        if op == "quantize":
            c = {"op": op, "rows": _log(rng, 1, 200000), "cin": _log(rng, 1, 8192), "dtype": rng.choice([F32, BF16, F16]), "pad": pad}
        elif op == "int8":
            c = {"op": op, "rows": _log(rng, 1, 100000), "cin": _log(rng, 16, 4200), "ctot": _log(rng, 2, 4200),
                 "dtype": rng.choice([F32, BF16, F16]), "act": rng.choice(["linear", "relu", "leaky_relu"]),
                 "bias": rng.random() < 0.5, "pad": pad}
        else:
            dtype = rng.choice([F32, BF16, F16])
            wide = op == "grouped" and dtype == F32
            groups = _log(rng, 1, 4000)
            split = "graphs" if wide or rng.random() < 0.4 else "experts"
            models = rng.randint(1, 46) if split == "graphs" else groups
            rows = groups * rng.randint(20, 300) if split == "graphs" else _log(rng, 1, 40000)
            c = {"op": op, "rows": rows, "cin": _log(rng, 4, 512 if wide else 2600), "ctot": _log(rng, 2, 512 if wide else 2600),
                 "dtype": dtype, "groups": groups, "models": models, "split": split,
                 "act": rng.choice(["linear", "relu", "leaky_relu"]), "bias": rng.random() < 0.5,
                 "layout": rng.randrange(1 << 30), "pad": pad}
            if models > 512:
                continue
        w = work(c)
        # float32 products are dearer for each operation than 8-bit ones
        dear = 8 if op == "grouped" and c["dtype"] == F32 else 2 if op == "grouped" else 1
        if w["bytes"] <= MAX_BYTES and w["flops"] * dear <= MAX_FLOPS:
            return c


# ---- sizes of a case ------------------------------------------------------------------------------------------------------------

def _sizes(case):
    """(rows of each group, model of each group or None): from the case alone."""
    rng = random.Random(case["layout"])
    G, rows = case["groups"], case["rows"]
    if case["split"] == "graphs":  # graphs within a factor of three of one another, models at random
        w = [rng.uniform(1.0, 3.0) for _ in range(G)]
        models = [rng.randrange(case["models"]) for _ in range(G)]
    else:  # experts: uneven, some without a row; expert g is model g
        w = [rng.expovariate(1.0) for _ in range(G)]
        models = None
    total, acc, ptr = sum(w), 0.0, [0]
    for x in w:
        acc += x
        ptr.append(min(rows, int(round(rows * acc / total))))
    ptr[-1] = rows
    return [b - a for a, b in zip(ptr, ptr[1:])], models


def work(case):
    op, rows, cin = case["op"], case["rows"], case["cin"]
    if op == "quantize":
        return {"bytes": rows * cin * (SIZE[case["dtype"]] + 1) + 4 * rows, "flops": 3 * rows * cin}
    ctot = case["ctot"]
    elem = SIZE[case["dtype"]] if op == "grouped" else 1
    used = 1
    if op != "int8":
        sizes, models = _sizes(case)
        models = range(len(sizes)) if models is None else models
        used = len({m for n, m in zip(sizes, models) if n})
    channel = (4 if op != "grouped" else 0) + (4 if case["bias"] else 0)
    b = rows * cin * elem + used * ctot * (cin * elem + channel) + rows * ctot * SIZE[case["dtype"]]
    if op != "grouped":
        b += 4 * rows
    return {"bytes": b, "flops": 2 * rows * cin * ctot}


# ---- inputs ---------------------------------------------------------------------------------------------------------------------

def _padded(x, pad):
    """The same values as a column slice of a matrix ``pad`` columns wider (rows at an odd stride)."""
    if not pad:
        return x
    wide = torch.zeros(x.shape[0], x.shape[1] + pad, dtype=x.dtype, device=x.device)
    wide[:, :x.shape[1]] = x
    return wide[:, :x.shape[1]]


def prepare(case, seed):
    dev = "cuda:0"
    gen = torch.Generator(device=dev).manual_seed(seed)
    rows, cin, op = case["rows"], case["cin"], case["op"]
    dtype = getattr(torch, case["dtype"])
    # activations behind a leaky relu, rows of different magnitude
    H = torch.randn(rows, cin, device=dev, generator=gen)
    H = torch.where(H > 0, H, LEAKY * H)
    H *= torch.exp(torch.randn(rows, 1, device=dev, generator=gen))
    state = {"op": op, "dtype": dtype, "act": case.get("act", "linear"), "bias": None}
    if op == "quantize":
        state["H"] = _padded(H.to(dtype), case["pad"])
        return state
    ctot, models = case["ctot"], case.get("models", 1)
    lim = (6.0 / (cin + ctot)) ** 0.5
    W = torch.empty(models, ctot, cin, device=dev).uniform_(-lim, lim, generator=gen)
    if case["bias"]:
        state["bias"] = torch.randn(models, ctot, device=dev, generator=gen) * 0.1
    if op == "grouped":
        state["H"], state["W"] = _padded(H.to(dtype), case["pad"]), W.to(dtype)
    else:
        hs = H.abs().amax(1).clamp_min(1e-30) / 127.0
        ws = W.abs().amax(2).clamp_min(1e-30) / 127.0
        state["H"] = _padded(torch.round(H / hs[:, None]).clamp_(-127, 127).to(torch.int8), case["pad"])
        state["W"] = torch.round(W / ws[:, :, None]).clamp_(-127, 127).to(torch.int8)
        state["hs"], state["ws"] = hs, ws
    if op == "int8":
        state["W"], state["ws"] = state["W"][0], state["ws"][0]
        if state["bias"] is not None:
            state["bias"] = state["bias"][0]
        return state
    sizes, of = _sizes(case)
    ptr = [0]
    for n in sizes:
        ptr.append(ptr[-1] + n)
    state["group_ptr"] = torch.tensor(ptr, dtype=torch.int32, device=dev)
    state["model_of_group"] = None if of is None else torch.tensor(of, dtype=torch.int32, device=dev)
    state["status"] = torch.zeros(1, dtype=torch.int32, device=dev)
    # the plain form's plan: which rows each model has (a slice where they lie together)
    blocks = {}
    for g, n in enumerate(sizes):
        if n:
            blocks.setdefault(g if of is None else of[g], []).append((ptr[g], ptr[g + 1]))
    state["rows_of"] = {m: slice(*b[0]) if len(b) == 1 else torch.cat([torch.arange(lo, hi, device=dev) for lo, hi in b])
                        for m, b in blocks.items()}
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------------------

def _act(y, act):
    if act == "relu":
        return torch.where(y > 0, y, torch.zeros_like(y))
    if act == "leaky_relu":
        return torch.where(y > 0, y, LEAKY * y)
    return y


def _plain(s):
    op = s["op"]
    if op == "quantize":
        x = s["H"].float()
        # both quotients in 64 bits: the scale is a float32 rounded once, and next to a half one step decides
        scale = (x.abs().amax(1).double() / 127.0).float().clamp_min(2.0 ** -126)
        q = torch.round(x.double() / scale.double()[:, None]).clamp(-127, 127).to(torch.int8)
        return {"q": q, "scale": scale}
    if op == "int8":
        y = s["H"].float() @ s["W"].float().t()
        y = y * s["hs"][:, None] * s["ws"]
        if s["bias"] is not None:
            y = y + s["bias"]
        return _act(y, s["act"]).to(s["dtype"])
    H, W = s["H"], s["W"]
    out = torch.empty(H.shape[0], W.shape[1], dtype=s["dtype"], device=H.device)
    for m, rows in s["rows_of"].items():
        y = H[rows].float() @ W[m].float().t()
        if op == "grouped_int8":
            y = y * s["hs"][rows][:, None] * s["ws"][m]
        if s["bias"] is not None:
            y = y + s["bias"][m]
        out[rows] = _act(y, s["act"]).to(s["dtype"])
    return out


def run(s):
    if not own:
        return _plain(s)
    eng, op = _eng(), s["op"]
    if op == "quantize":
        q, scale = eng.quantize_rows(s["H"])
        return {"q": q, "scale": scale}
    if op == "int8":
        return eng.transform_int8(s["H"], s["hs"], s["W"], s["ws"], bias=s["bias"], act=s["act"], dtype=s["dtype"])
    if op == "grouped":
        return eng.transform_grouped(s["H"], s["W"], s["group_ptr"], model_of_group=s["model_of_group"], bias=s["bias"], act=s["act"],
                                     status=s["status"])
    return eng.transform_grouped_int8(s["H"], s["hs"], s["W"], s["ws"], s["group_ptr"], model_of_group=s["model_of_group"],
                                      bias=s["bias"], act=s["act"], dtype=s["dtype"], status=s["status"])


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    H = s["H"].to(torch.float64)
    if s["op"] == "quantize":
        # the scale is a float32 by definition: the quotient is taken by the value that is stored
        largest = torch.linalg.vector_norm(H, ord=float("inf"), dim=1)
        scale = torch.maximum(largest / 127, torch.full_like(largest, 2.0 ** -126)).to(torch.float32)
        steps = torch.round(torch.div(H, scale.to(torch.float64).unsqueeze(1)))
        return {"q": steps.clamp(-127, 127).to(torch.int8), "scale": largest / 127}
    if s["op"] != "grouped":
        H = H * s["hs"].to(torch.float64).unsqueeze(1)
    if s["op"] == "int8":
        groups = [(0, case["rows"], 0)]
        W, ws, bias = s["W"][None], s["ws"][None], s["bias"][None] if case["bias"] else None
    else:
        sizes, of = _sizes(case)
        W, ws, bias = s["W"], s.get("ws"), s["bias"]
        groups, at = [], 0
        for g, n in enumerate(sizes):
            groups.append((at, at + n, g if of is None else of[g]))
            at += n
    y = torch.zeros(case["rows"], case["ctot"], dtype=torch.float64, device=H.device)
    for lo, hi, m in groups:
        if hi > lo:
            weights = W[m].to(torch.float64)
            if ws is not None:
                weights = weights * ws[m].to(torch.float64).unsqueeze(1)
            y[lo:hi] = torch.mm(H[lo:hi], weights.t())
            if bias is not None:
                y[lo:hi] += bias[m].to(torch.float64)
    if case["act"] == "relu":
        y.clamp_min_(0)
    elif case["act"] == "leaky_relu":
        y = torch.maximum(y, y * LEAKY)
    return y
