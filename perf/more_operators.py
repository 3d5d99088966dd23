"""What a transformer's training step needs beside its products and norms, as cases that can be timed and compared.

Four kinds, each one pass through an operator that a step calls:

    gated_fwd   a gated Linear layer: y = act(x Wg^T + bg) * (x Wu^T + bu), and what its backward reads
    gated_bwd   its gradients with respect to x, W = [Wg; Wu] and b = [bg; bu], from the kept projections
    rotary      rotation of queries and keys by their positions, along one axis or several (time, height, width)
    clip        the global norm of many gradients, and the gradients scaled down to a largest norm
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
CODE = {"f32": 0, "f16": 1, "bf16": 2}
POSITIONS = {"i32": (torch.int32, 4, 3), "i64": (torch.int64, 8, 4)}
GATE = {"silu": 0, "gelu_tanh": 2, "sigmoid": 3, "relu": 4}


# --------------------------------------------------------------------------- #
# The cases
# --------------------------------------------------------------------------- #


def listed():
    """gated: `keep`, whether the projections are kept for a backward pass.  rotary: `axes` positions a token; the pairs of a head's
    first `rotated` columns belong to the axes in "runs" or in "turns" and are "halves" (i, i + rotated / 2) or "neighbours"
    (2 i, 2 i + 1); `packed`: queries and keys as they lie in one (B, S, 3, H, D) tensor; `inverse`: as in the backward pass."""
    return [
        # One token of the character-level transformer, when it writes text: the launch is what counts.
        {"name": "gated_fwd_token", "kind": "gated_fwd", "dtype": "bf16", "rows": 1, "inputs": 384, "outputs": 1024,
         "gate": "silu", "bias": False, "keep": False},
        # A few sequences that are continued by a wide model, a token each: the weights are what counts.
        {"name": "gated_fwd_tokens", "kind": "gated_fwd", "dtype": "bf16", "rows": 8, "inputs": 4096, "outputs": 8192,
         "gate": "silu", "bias": False, "keep": False},
        # The character-level transformer at the size it is trained at: 64 sequences of 256 tokens.
        {"name": "gated_fwd_char", "kind": "gated_fwd", "dtype": "bf16", "rows": 16384, "inputs": 384, "outputs": 1024,
         "gate": "silu", "bias": False, "keep": True},
        # A layer of a large model in training, where the matrix cores are all that counts.
        {"name": "gated_fwd_large", "kind": "gated_fwd", "dtype": "bf16", "rows": 8192, "inputs": 4096, "outputs": 8192,
         "gate": "silu", "bias": False, "keep": True},
        # The gradients of a batch and widths that are multiples of nothing.
        {"name": "gated_bwd_ragged", "kind": "gated_bwd", "dtype": "f16", "rows": 1999, "inputs": 767, "outputs": 1001,
         "gate": "gelu_tanh", "bias": True},
        # The character-level transformer's.
        {"name": "gated_bwd_char", "kind": "gated_bwd", "dtype": "bf16", "rows": 16384, "inputs": 384, "outputs": 1024,
         "gate": "silu", "bias": False},
        # A layer in fp32, the rows and inputs of the fp32 classifier's.
        {"name": "gated_bwd_f32", "kind": "gated_bwd", "dtype": "f32", "rows": 2048, "inputs": 784, "outputs": 512,
         "gate": "gelu_tanh", "bias": True},
        # One new token of each of 32 sequences, far into them; only half of a head's columns turn.
        {"name": "rotary_token", "kind": "rotary", "dtype": "f16", "batch": 32, "length": 1, "heads": 32, "columns": 128,
         "rotated": 64, "axes": 1, "order": "runs", "pairs": "halves", "packed": False, "inverse": False, "far": 1000000,
         "positions": "i64"},
        # Queries and keys of the character-level transformer in its packed projection.
        {"name": "rotary_char", "kind": "rotary", "dtype": "bf16", "batch": 64, "length": 256, "heads": 6, "columns": 64,
         "rotated": 64, "axes": 1, "order": "runs", "pairs": "halves", "packed": True, "inverse": False, "far": 0,
         "positions": "i32"},
        # The gradient of the queries of a clip of video: 32 frames of 32 x 32 patches.
        {"name": "rotary_video", "kind": "rotary", "dtype": "bf16", "batch": 1, "length": 32768, "heads": 32, "columns": 128,
         "rotated": 128, "axes": 3, "order": "runs", "pairs": "halves", "packed": False, "inverse": True, "far": 0,
         "positions": "i32"},
        # The fp32 gradients of the character-level transformer, a tensor a parameter.
        {"name": "clip_char", "kind": "clip", "dtype": "f32", "tensors": 68, "elements": 10750000, "aligned": True, "share": 0.25},
        # 16-bit gradients of a larger model, packed without gaps.
        {"name": "clip_large", "kind": "clip", "dtype": "bf16", "tensors": 290, "elements": 300000000, "aligned": False, "share": 0.5},
    ]


def _between(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo, hi):
    """A feature count: as a rule a multiple of 8, now and then any number."""
    n = _between(rng, lo, hi)
    return n if rng.random() < 0.25 else max(lo, n // 8 * 8)


def _draw(rng):
    kind = rng.choice(["gated_fwd", "gated_fwd", "gated_bwd", "gated_bwd", "rotary", "clip"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("gated_fwd", "gated_bwd"):
        case = {"kind": kind, "dtype": dtype, "rows": _between(rng, 1 if kind == "gated_fwd" else 16, 32768),
                "inputs": _width(rng, 32, 8192), "outputs": _width(rng, 32, 16384), "gate": rng.choice(sorted(GATE)),
                "bias": rng.random() < 0.4}
        if kind == "gated_fwd":
            case["keep"] = rng.random() < 0.6
        return case
    if kind == "rotary":
        columns = rng.choice([32, 64, 64, 80, 96, 128, 128, 256, 66, 50])
        axes = rng.choice([1, 1, 2, 3])
        return {"kind": kind, "dtype": dtype, "batch": _between(rng, 1, 64), "length": _between(rng, 1, 32768),
                "heads": _between(rng, 1, 64), "columns": columns, "rotated": rng.choice([columns, columns, columns // 4 * 2]),
                "axes": axes, "order": rng.choice(["runs", "turns"]), "pairs": rng.choice(["halves", "halves", "neighbours"]),
                "packed": rng.random() < 0.4, "inverse": rng.random() < 0.5, "far": rng.choice([0, 0, 5000, 1000000]),
                "positions": rng.choice(["i32", "i64"])}
    tensors = _between(rng, 1, 400)
    return {"kind": kind, "dtype": dtype, "tensors": tensors, "elements": max(tensors, _between(rng, 100, 300000000)),
            "aligned": rng.random() < 0.6, "share": rng.choice([0.01, 0.5, 0.9, 2.0])}


def _seconds(case):
    w = work(case)
    return max(w["flops"] / (1e14 if case["dtype"] == "f32" else 1e15), w["bytes"] / 4e12)


def draw(rng):
    """One more case: as `_draw` spreads them, of those that take no longer than the largest listed ones."""
    most = {}
    for case in listed():
        kind = case["kind"][:5]  # (both passes of a gated layer cost at most what the largest of them does)
        most[kind] = max(most.get(kind, 0.0), _seconds(case))
    while True:
        case = _draw(rng)
        if _seconds(case) <= most[case["kind"][:5]]:
            return case


def work(case):
    s = SIZE[case["dtype"]]
    if case["kind"] in ("gated_fwd", "gated_bwd"):
        M, K, F = case["rows"], case["inputs"], case["outputs"]
        bias = 2 * F if case["bias"] else 0
        if case["kind"] == "gated_fwd":
            return {"bytes": s * (M * K + 2 * F * K + bias + M * F * (3 if case["keep"] else 1)), "flops": 4 * M * F * K}
        return {"bytes": s * (3 * M * F + 2 * M * K + 4 * F * K + bias), "flops": 8 * M * F * K}
    if case["kind"] == "rotary":
        tokens, heads = case["batch"] * case["length"], case["heads"] * (2 if case["packed"] else 1)
        n = tokens * heads * case["columns"]
        return {"bytes": 2 * n * s + tokens * case["axes"] * POSITIONS[case["positions"]][1],
                "flops": 3 * tokens * heads * case["rotated"]}
    return {"bytes": 3 * case["elements"] * s, "flops": 3 * case["elements"]}


def _axis_of_pairs(case):
    """The axis that each pair of columns turns by: one run of pairs an axis, or the axes in turn."""
    pairs, axes = case["rotated"] // 2, case["axes"]
    if case["order"] == "turns":
        return [i % axes for i in range(pairs)]
    return [min(i * axes // pairs, axes - 1) for i in range(pairs)]


def _places(case):
    """Where the tensors of a clip case lie in the flat array: (first element, elements) of each, of very different sizes."""
    count, total = case["tensors"], case["elements"]
    weights = [1 if i % 3 == 2 else 1000 + i * 7919 % 4096 for i in range(count)]
    whole, at, places, given, upto = sum(weights), 0, [], 0, 0
    for w in weights:
        upto += w
        n = max(1, upto * total // whole - given)
        places.append((at, n))
        given += n
        at += -(-n // 64) * 64 if case["aligned"] else n
    return places, at


# --------------------------------------------------------------------------- #
# Inputs
# --------------------------------------------------------------------------- #


def _inputs(case, seed):
    """What both the program and the check take: tensors from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = TYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    if case["kind"] in ("gated_fwd", "gated_bwd"):
        M, K, F = case["rows"], case["inputs"], case["outputs"]
        # what a norm puts out, columns of different size; weights that keep that size
        x = normal(M, K) * torch.exp(0.5 * normal(K))
        s = {"x": x.to(t), "w": (normal(2 * F, K) * (1.3 * K) ** -0.5).to(t)}
        if case["kind"] == "gated_fwd":
            s["bias"] = (0.2 * normal(2 * F)).to(t) if case["bias"] else None
            return s
        s["gu"] = (1.2 * normal(M, 2 * F)).to(t)
        s["dy"] = (0.5 * normal(M, F)).to(t)  # (as the loss is scaled for fp16)
        return s
    if case["kind"] == "rotary":
        B, S, H, D = case["batch"], case["length"], case["heads"], case["columns"]
        x = (normal(B, S, 3 * H if case["packed"] else H, D) * torch.exp(0.5 * normal(D))).to(t)
        pairs = case["rotated"] // 2
        exponent = torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs
        first = case["far"] + torch.randint(0, 64, (case["axes"], B, 1), generator=g, device="cuda")
        at = torch.arange(S, device="cuda")
        side = max(1, math.isqrt(max(1, S // 32)))
        steps = [at] if case["axes"] == 1 else [at // (side * side), at // side % side, at % side][3 - case["axes"]:]
        return {"x": x, "inv_freq": torch.pow(10000.0, -exponent).float(),
                "positions": (first + torch.stack(steps)[:, None, :]).to(POSITIONS[case["positions"]][0])}
    places, flat = _places(case)
    grads = torch.zeros(flat, dtype=t, device="cuda")
    square = 0.0
    for at, n in places:
        size = 0.02 / (1 + at % 7)
        grads[at:at + n] = (size * normal(n)).to(t)
        square += size * size * n
    return {"grads": grads, "max_norm": case["share"] * math.sqrt(square)}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    t = TYPES[case["dtype"]]
    empty = lambda *shape, dtype=t: torch.empty(*shape, dtype=dtype, device="cuda")
    # the buffers that the program has for the results, and what it says of its tensors
    if case["kind"] == "gated_fwd":
        M, F = case["rows"], case["outputs"]
        s["out"] = {"y": empty(M, F), "gu": empty(M, 2 * F) if case["keep"] else None}
    elif case["kind"] == "gated_bwd":
        M, K, F = case["rows"], case["inputs"], case["outputs"]
        s["out"] = {"dx": empty(M, K), "dw": empty(2 * F, K), "db": empty(2 * F) if case["bias"] else None}
    elif case["kind"] == "rotary":
        B, S, D = case["batch"], case["length"], case["columns"]
        heads = case["heads"] * (2 if case["packed"] else 1)  # queries and keys, without the values behind them
        s["out"] = {"y": empty(B, S, heads, D)}
        pairs = case["rotated"] // 2
        s["heads"], s["pair_axis"] = heads, (ctypes.c_int32 * pairs)(*_axis_of_pairs(case))
        strides = lambda v: (ctypes.c_int64 * 3)(*v.stride()[:3])
        s["strides"] = strides(s["x"]), strides(s["out"]["y"]), strides(s["positions"])
        s["axis"] = torch.tensor(_axis_of_pairs(case), device="cuda")
    else:
        places, flat = _places(case)
        out = torch.zeros(flat, dtype=t, device="cuda")
        s["out"] = {"norm": empty(1, dtype=torch.float32), "grads": out}
        n = len(places)
        pointers = lambda v: (ctypes.c_void_p * n)(*[v.data_ptr() + at * v.element_size() for at, _ in places])
        s["tensors"] = (n, pointers(s["grads"]), pointers(out), (ctypes.c_int64 * n)(*[k for _, k in places]),
                        (ctypes.c_int * n)(*[CODE[case["dtype"]]] * n))
    return s


# --------------------------------------------------------------------------- #
# One pass
# --------------------------------------------------------------------------- #


def run(s):
    if own:
        return _run_own(s)
    return {"gated_fwd": _plain_gated_fwd, "gated_bwd": _plain_gated_bwd, "rotary": _plain_rotary, "clip": _plain_clip}[s["case"]["kind"]](s)


def _run_own(s):
    import mograd_amd

    case, lib, out = s["case"], mograd_amd.load(), s["out"]
    code = CODE[case["dtype"]]
    stream = torch.cuda.current_stream().cuda_stream
    p = lambda t: None if t is None else t.data_ptr()
    if case["kind"] == "gated_fwd":
        lib.mg_gated_linear_fwd(p(s["x"]), p(s["w"]), p(s["bias"]), p(out["y"]), p(out["gu"]), case["rows"], case["outputs"],
                                case["inputs"], GATE[case["gate"]], code, stream)
    elif case["kind"] == "gated_bwd":
        lib.mg_gated_linear_bwd(p(s["dy"]), p(s["gu"]), p(s["x"]), p(s["w"]), p(out["dx"]), p(out["dw"]), p(out["db"]), case["rows"],
                                case["outputs"], case["inputs"], 0, GATE[case["gate"]], code, code, stream)
    elif case["kind"] == "rotary":
        x_strides, y_strides, pos_strides = s["strides"]
        lib.mg_rotary(p(s["x"]), p(out["y"]), p(s["positions"]), p(s["inv_freq"]), s["pair_axis"], case["batch"], case["length"],
                      s["heads"], case["columns"], case["rotated"], x_strides, y_strides, pos_strides, case["axes"],
                      POSITIONS[case["positions"]][2], int(case["pairs"] == "neighbours"), int(case["inverse"]), code, stream)
    else:
        count, grads, clipped, numels, dtypes = s["tensors"]
        lib.mg_clip_grads(grads, clipped, numels, dtypes, count, s["max_norm"], p(out["norm"]), stream)
    return out


def _plain_gate(g, kind):
    """act(g) and its derivative."""
    if kind == "relu":
        on = (g > 0).float()
        return g * on, on
    if kind == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        z = 2 * c * (g + 0.044715 * g * g * g)
        s = 1 / (1 + torch.exp(-z))
        return g * s, s + g * s * (1 - s) * 2 * c * (1 + 3 * 0.044715 * g * g)
    s = 1 / (1 + torch.exp(-g))
    if kind == "sigmoid":
        return s, s * (1 - s)
    return g * s, s * (1 + g * (1 - s))


def _plain_gated_fwd(s):
    case = s["case"]
    t, F = TYPES[case["dtype"]], case["outputs"]
    gu = s["x"].float() @ s["w"].float().t()
    if case["bias"]:
        gu += s["bias"].float()
    y = (_plain_gate(gu[:, :F], case["gate"])[0] * gu[:, F:]).to(t)
    return {"y": y, "gu": gu.to(t) if case["keep"] else None}


def _plain_gated_bwd(s):
    case = s["case"]
    t, F = TYPES[case["dtype"]], case["outputs"]
    gu, dy = s["gu"].float(), s["dy"].float()
    act, slope = _plain_gate(gu[:, :F], case["gate"])
    d = torch.cat([dy * gu[:, F:] * slope, dy * act], dim=1)
    return {"dx": (d @ s["w"].float()).to(t), "dw": (d.t() @ s["x"].float()).to(t), "db": d.sum(dim=0).to(t) if case["bias"] else None}


def _plain_rotary(s):
    case, R = s["case"], s["case"]["rotated"]
    # angles of far positions lose their fraction of a turn in 32 bits
    angle = s["positions"].double()[s["axis"]].permute(1, 2, 0) * s["inv_freq"].double()
    if case["inverse"]:
        angle = -angle
    cos, sin = torch.cos(angle).float()[:, :, None, :], torch.sin(angle).float()[:, :, None, :]
    x = s["x"][:, :, :s["heads"]]
    y = x.clone()
    first, second = (slice(0, R, 2), slice(1, R, 2)) if case["pairs"] == "neighbours" else (slice(0, R // 2), slice(R // 2, R))
    a, b = x[..., first].float(), x[..., second].float()
    y[..., first] = (a * cos - b * sin).to(y.dtype)
    y[..., second] = (a * sin + b * cos).to(y.dtype)
    return {"y": y}


def _plain_clip(s):
    """(Between the tensors there are zeros, which add nothing.)"""
    g = s["grads"]
    norm = torch.sqrt(g.double().square().sum()).float().reshape(1)
    scale = torch.where(norm > s["max_norm"], s["max_norm"] / norm, 1.0)
    return {"norm": norm, "grads": (g.float() * scale).to(g.dtype)}


# --------------------------------------------------------------------------- #
# The same from the definitions, in 64 bits
# --------------------------------------------------------------------------- #


def exact(case, seed):
    s = _inputs(case, seed)
    return {"gated_fwd": _exact_gated_fwd, "gated_bwd": _exact_gated_bwd, "rotary": _exact_rotary, "clip": _exact_clip}[case["kind"]](case, s)


def _exact_gate(g, kind):
    """act(g) = g P(g) or P(g), and its derivative from P and P'."""
    if kind == "relu":
        p = torch.heaviside(g, torch.zeros_like(g))
        return g * p, p
    if kind == "gelu_tanh":
        k = (2 / math.pi) ** 0.5
        th = torch.tanh(k * g * (1 + 0.044715 * g ** 2))
        p, dp = 0.5 * (1 + th), 0.5 * (1 - th ** 2) * k * (1 + 0.134145 * g ** 2)
        return g * p, p + g * dp
    p = torch.sigmoid(g)
    dp = p * torch.sigmoid(-g)
    return (p, dp) if kind == "sigmoid" else (g * p, p + g * dp)


def _exact_gated_fwd(case, s):
    F = case["outputs"]
    x = s["x"].double()
    part = lambda i: torch.matmul(x, s["w"][i * F:(i + 1) * F].double().t()) + (s["bias"][i * F:(i + 1) * F].double() if case["bias"] else 0.0)
    g, u = part(0), part(1)
    y = _exact_gate(g, case["gate"])[0] * u
    return {"y": y, "gu": torch.cat([g, u], dim=1) if case["keep"] else None}


def _exact_gated_bwd(case, s):
    """The gradients of the two projections on their own, each from its definition."""
    F = case["outputs"]
    x, dy = s["x"].double(), s["dy"].double()
    act, slope = _exact_gate(s["gu"][:, :F].double(), case["gate"])
    dg, du = slope.mul_(s["gu"][:, F:].double()).mul_(dy), act.mul_(dy)
    dx = torch.matmul(dg, s["w"][:F].double()) + torch.matmul(du, s["w"][F:].double())
    dw = torch.cat([torch.matmul(d.t().contiguous(), x) for d in (dg, du)])
    ones = torch.ones(case["rows"], dtype=torch.float64, device="cuda")
    return {"dx": dx, "dw": dw, "db": torch.cat([torch.matmul(ones, dg), torch.matmul(ones, du)]) if case["bias"] else None}


def _exact_rotary(case, s):
    """Each pair of columns as a complex number, turned by its angle."""
    heads, pairs = case["heads"] * (2 if case["packed"] else 1), case["rotated"] // 2
    out = s["x"][:, :, :heads].double()
    sign = -1.0 if case["inverse"] else 1.0
    for i, axis in enumerate(_axis_of_pairs(case)):
        turn = sign * s["positions"][axis].double() * s["inv_freq"][i].double()
        turn = torch.polar(torch.ones_like(turn), turn)[:, :, None]
        a, b = (2 * i, 2 * i + 1) if case["pairs"] == "neighbours" else (i, i + pairs)
        z = torch.complex(out[..., a], out[..., b]) * turn
        out[..., a], out[..., b] = z.real, z.imag
    return {"y": out}


def _exact_clip(case, s):
    """Tensor by tensor."""
    places, flat = _places(case)
    square = sum(float(torch.dot(v, v)) for v in (s["grads"][at:at + n].double() for at, n in places))
    norm = math.sqrt(square)
    out = torch.zeros(flat, dtype=torch.float64, device="cuda")
    for at, n in places:
        out[at:at + n] = s["grads"][at:at + n].double() * min(1.0, s["max_norm"] / norm)
    return {"norm": torch.tensor([norm], dtype=torch.float64, device="cuda"), "grads": out}
