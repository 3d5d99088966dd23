"""The residual path of a transformer block in training, and its activations in 8 bits, as cases that can be timed and compared.

Four kinds, each one pass through the operators that a training step calls:

    norm_fwd   between two blocks: the block's output f is normalised, gated and added to the scaled residual stream h, and the
               sum is normalised for the next block
    norm_bwd   the gradients of that, from the saved statistics, with f as it was or as it is kept in 8 bits
    act8       an activation put away in 8 bits and brought back
    linear     the three gradients of a Linear layer whose input was kept in 8 bits

Activations in 8 bits ("act8"): blocks of 32 columns of a row (the last one may be shorter) share a power of two 2^k, the least
one for which the block's values are whole numbers of at most 127 after rounding; a value is kept as that whole number q.
One run of bytes holds them: rows x ld bytes of q, ld the columns rounded up to 32 (zeros past the columns), then rows x ld / 32
bytes of k + 133.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
CODE = {"f32": 0, "f16": 1, "bf16": 2}
K_RANGE = {"f32": (-126, 121), "f16": (-24, 9), "bf16": (-126, 121)}
EPS = 1e-5
BLOCK = 32


# --------------------------------------------------------------------------- #
# The cases
# --------------------------------------------------------------------------- #


def listed():
    """gate: "none", "channel" (one number a column) or "sequence" (one vector for every `gate_rows` rows)."""
    return [
        # A first experiment: 4 sequences of 32 tokens, 64 wide, fp32. What a user waits for is the launch.
        {"name": "norm_fwd_toy", "kind": "norm_fwd", "dtype": "f32", "rows": 128, "cols": 64, "gate": "channel",
         "gate_rows": 128, "post": True, "pre": True, "scale": 1.0},
        # The character-level transformer at the size it is trained at: 64 sequences of 256 tokens.
        {"name": "norm_fwd_char", "kind": "norm_fwd", "dtype": "bf16", "rows": 16384, "cols": 384, "gate": "channel",
         "gate_rows": 16384, "post": True, "pre": True, "scale": 1.0},
        # A wide model's stream, a gate for each of 8 sequences that a conditioning network has made.
        {"name": "norm_fwd_wide", "kind": "norm_fwd", "dtype": "bf16", "rows": 8192, "cols": 4096, "gate": "sequence",
         "gate_rows": 1024, "post": True, "pre": True, "scale": 0.875},
        # A batch and a width that are multiples of nothing.
        {"name": "norm_bwd_ragged", "kind": "norm_bwd", "dtype": "f16", "rows": 2587, "cols": 1001, "gate": "sequence",
         "gate_rows": 199, "post": True, "pre": True, "scale": 0.75, "f8": False, "grads": "f16"},
        # The character-level transformer, f kept in 8 bits, fp32 gradients of the parameters.
        {"name": "norm_bwd_char", "kind": "norm_bwd", "dtype": "bf16", "rows": 16384, "cols": 384, "gate": "channel",
         "gate_rows": 16384, "post": True, "pre": True, "scale": 1.0, "f8": True, "grads": "f32"},
        # fp32 rows of 4096 columns, the size of the framework's LayerNorm benchmark.
        {"name": "norm_bwd_f32", "kind": "norm_bwd", "dtype": "f32", "rows": 2048, "cols": 4096, "gate": "channel",
         "gate_rows": 2048, "post": True, "pre": True, "scale": 1.0, "f8": False, "grads": "f32"},
        # What the transformer's ReLU puts out: half of it zeros, and signs that have to stay.
        {"name": "act8_char", "kind": "act8", "dtype": "bf16", "rows": 16384, "cols": 1536, "relu": True},
        # A small batch of odd width.
        {"name": "act8_ragged", "kind": "act8", "dtype": "f16", "rows": 333, "cols": 1001, "relu": False},
        # The transformer's second feed-forward product, the ReLU's gradient on its dX.
        {"name": "linear_char", "kind": "linear", "dtype": "bf16", "rows": 16384, "inputs": 1536, "outputs": 384,
         "relu": True, "bias": False, "grads": "f32"},
        # A small layer whose batch and widths are odd.
        {"name": "linear_ragged", "kind": "linear", "dtype": "f16", "rows": 1999, "inputs": 768, "outputs": 1001,
         "relu": False, "bias": True, "grads": "f16"},
        # A layer of a large model, where the matrix cores are all that counts.
        {"name": "linear_large", "kind": "linear", "dtype": "bf16", "rows": 8192, "inputs": 4096, "outputs": 4096,
         "relu": False, "bias": False, "grads": "bf16"},
        # The fp32 classifier's layer.
        {"name": "linear_f32", "kind": "linear", "dtype": "f32", "rows": 2048, "inputs": 784, "outputs": 512,
         "relu": True, "bias": True, "grads": "f32"},
    ]


def _between(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo, hi):
    """A feature count: as a rule a multiple of 8, now and then any number."""
    n = _between(rng, lo, hi)
    return n if rng.random() < 0.25 else max(lo, n // 8 * 8)


def _draw(rng):
    kind = rng.choice(["norm_fwd", "norm_bwd", "norm_bwd", "act8", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("norm_fwd", "norm_bwd"):
        gate = rng.choice(["none", "channel", "sequence"])
        post = rng.random() < 0.8
        cols = _width(rng, 32, 8192)
        if gate == "sequence":
            sequences, length = _between(rng, 1, 64), _between(rng, 16, 2048)
            rows, gate_rows = sequences * length, length
        else:
            rows = gate_rows = _between(rng, 1, 65536)
        case = {"kind": kind, "dtype": dtype, "rows": rows, "cols": cols, "gate": gate, "gate_rows": gate_rows, "post": post,
                "pre": rng.random() < 0.8 or not post, "scale": rng.choice([1.0, 1.0, 0.5, 1.25])}
        if kind == "norm_bwd":
            case["f8"] = rng.random() < 0.5
            case["grads"] = rng.choice(["f32", dtype])
        return case
    if kind == "act8":
        return {"kind": kind, "dtype": dtype, "rows": _between(rng, 1, 65536), "cols": _width(rng, 32, 8192),
                "relu": rng.random() < 0.5}
    return {"kind": kind, "dtype": dtype, "rows": _between(rng, 16, 32768), "inputs": _width(rng, 32, 8192),
            "outputs": _width(rng, 32, 8192), "relu": rng.random() < 0.5, "bias": rng.random() < 0.5,
            "grads": rng.choice(["f32", dtype])}


def _seconds(case):
    w = work(case)
    return max(w["flops"] / (1e14 if case["dtype"] == "f32" else 1e15), w["bytes"] / 4e12)


def draw(rng):
    """One more case: as `_draw` spreads them, of those that take no longer than the largest listed ones."""
    most = {}
    for case in listed():
        most[case["kind"]] = max(most.get(case["kind"], 0.0), _seconds(case))
    while True:
        case = _draw(rng)
        if _seconds(case) <= most[case["kind"]]:
            return case


def _act8_bytes(rows, cols):
    ld = -(-cols // BLOCK) * BLOCK
    return rows * (ld + ld // BLOCK)


def work(case):
    s = SIZE[case["dtype"]]
    if case["kind"] == "act8":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * s + 2 * _act8_bytes(case["rows"], case["cols"]), "flops": 4 * n}
    if case["kind"] == "linear":
        M, K, N = case["rows"], case["inputs"], case["outputs"]
        g = SIZE[case["grads"]]
        return {"bytes": s * (M * N + N * K + M * K) + _act8_bytes(M, K) + g * (N * K + (N if case["bias"] else 0)),
                "flops": 4 * M * N * K + (M * N if case["bias"] else 0)}
    rows, cols = case["rows"], case["cols"]
    n = rows * cols
    stats = 8 * rows * (case["post"] + case["pre"])
    gates = {"none": 0, "channel": 1, "sequence": rows // case["gate_rows"]}[case["gate"]]
    params = gates + 2 * case["post"] + 2 * case["pre"]
    if case["kind"] == "norm_fwd":
        return {"bytes": n * s * (3 + case["pre"]) + stats + params * cols * s, "flops": n * (4 + 8 * case["post"] + 8 * case["pre"])}
    f = _act8_bytes(rows, cols) if case["f8"] else n * s
    return {"bytes": n * s * (3 + 2 * case["pre"]) + f + stats + cols * ((params - case["pre"]) * s + params * SIZE[case["grads"]]),
            "flops": n * (6 + 12 * case["post"] + 12 * case["pre"])}


# --------------------------------------------------------------------------- #
# Activations in 8 bits, in plain operations
# --------------------------------------------------------------------------- #


def _act8_parts(act8, rows, cols):
    """q (rows, blocks, 32) and k (rows, blocks) of a run of bytes."""
    blocks = -(-cols // BLOCK)
    q = act8[:rows * blocks * BLOCK].view(torch.int8).view(rows, blocks, BLOCK)
    k = act8[rows * blocks * BLOCK:].view(rows, blocks).to(torch.int32) - 133
    return q, k


def _power(k):
    """2^k in fp32, -126 <= k <= 127."""
    return (k + 127 << 23).to(torch.int32).view(torch.float32)


def _act8_store(x, dtype, keep_sign):
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    v = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - cols)).view(rows, blocks, BLOCK)
    part, power = torch.frexp(v.abs().amax(dim=2))
    k = power - 7 + (part >= 127.5 / 128).to(power.dtype)
    k = torch.where(part > 0, k, K_RANGE[dtype][0]).clamp(*K_RANGE[dtype])
    q = torch.round(v * _power(-k)[:, :, None]).clamp(-127, 127)
    if keep_sign:
        q = torch.where(q == 0, torch.sign(v), q)
    act8 = torch.empty(_act8_bytes(rows, cols), dtype=torch.uint8, device=x.device)
    act8[:v.numel()] = q.to(torch.int8).reshape(-1).view(torch.uint8)
    act8[v.numel():] = (k + 133).to(torch.uint8).reshape(-1)
    return act8


def _act8_load(act8, rows, cols):
    q, k = _act8_parts(act8, rows, cols)
    return (q.float() * _power(k)[:, :, None]).view(rows, -1)[:, :cols]


# --------------------------------------------------------------------------- #
# Inputs
# --------------------------------------------------------------------------- #


def _activations(g, rows, cols, dtype, spread=1.0, offset=0.0):
    """Normal values whose columns differ in size, a few of them by much, as activations' do."""
    size = torch.exp(0.5 * torch.randn(cols, generator=g, device="cuda"))
    size = torch.where(torch.rand(cols, generator=g, device="cuda") < 0.01, size * 12, size)
    x = torch.randn(rows, cols, generator=g, device="cuda") * size * spread + offset
    return x.to(TYPES[dtype])


def _statistics(x):
    mean = torch.empty(x.shape[0], device=x.device)
    rstd = torch.empty(x.shape[0], device=x.device)
    for i in range(0, x.shape[0], 4096):
        v = x[i:i + 4096].double()
        m = v.mean(dim=1)
        mean[i:i + 4096] = m.float()
        rstd[i:i + 4096] = torch.rsqrt((v - m[:, None]).square().mean(dim=1) + EPS).float()
    return mean, rstd


def _seeded(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _inputs(case, seed):
    """What both the program and the check take: tensors from the seed alone."""
    g = _seeded(seed)
    dtype = case["dtype"]
    t = TYPES[dtype]
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    if case["kind"] == "act8":
        x = _activations(g, case["rows"], case["cols"], dtype)
        return {"x": torch.relu(x) if case["relu"] else x}
    if case["kind"] == "linear":
        M, K, N = case["rows"], case["inputs"], case["outputs"]
        x = _activations(g, M, K, dtype)
        x8 = _act8_store(torch.relu(x) if case["relu"] else x, dtype, case["relu"])
        return {"dy": (normal(M, N) * 0.05).to(t), "x8": x8, "w": (normal(N, K) * K ** -0.5).to(t)}
    rows, cols = case["rows"], case["cols"]
    gates = {"none": 0, "channel": 1, "sequence": rows // case["gate_rows"]}[case["gate"]]
    s = {"f": _activations(g, rows, cols, dtype), "gate": (0.5 + 0.3 * normal(gates, cols)).to(t) if gates else None}
    for norm in ("post", "pre"):
        s[norm + "_gamma"] = (1 + 0.25 * normal(cols)).to(t) if case[norm] else None
        s[norm + "_beta"] = (0.1 * normal(cols)).to(t) if case[norm] else None
    # the stream: wider than what a block adds to it, and not centred
    h = _activations(g, rows, cols, dtype, 2.0, 0.5)
    if case["kind"] == "norm_fwd":
        s["h"] = h
        return s
    s["h_out"] = h
    s["dh_out"] = (normal(rows, cols) * 0.05).to(t)
    s["dx"] = (normal(rows, cols) * 0.05).to(t) if case["pre"] else None
    s["post_mean"], s["post_rstd"] = _statistics(s["f"]) if case["post"] else (None, None)
    s["pre_mean"], s["pre_rstd"] = _statistics(h) if case["pre"] else (None, None)
    if case["f8"]:
        s["f8"] = _act8_store(s["f"], dtype, False)
        s["f"] = None
    else:
        s["f8"] = None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        import mograd_amd

        s["lib"] = mograd_amd.load()
        s["out"] = _outputs(case)
    return s


def _outputs(case):
    """The buffers that the program has for the results."""
    t = TYPES[case["dtype"]]
    empty = lambda *shape, dtype=t: torch.empty(*shape, dtype=dtype, device="cuda")
    if case["kind"] == "act8":
        return {"act8": empty(_act8_bytes(case["rows"], case["cols"]), dtype=torch.uint8), "x": empty(case["rows"], case["cols"])}
    if case["kind"] == "linear":
        M, K, N = case["rows"], case["inputs"], case["outputs"]
        g = TYPES[case["grads"]]
        return {"dx": empty(M, K), "dw": empty(N, K, dtype=g), "db": empty(N, dtype=g) if case["bias"] else None}
    rows, cols = case["rows"], case["cols"]
    if case["kind"] == "norm_fwd":
        out = {"h_out": empty(rows, cols), "x": empty(rows, cols) if case["pre"] else None}
        for norm in ("post", "pre"):
            for stat in ("mean", "rstd"):
                out[f"{norm}_{stat}"] = empty(rows, dtype=torch.float32) if case[norm] else None
        return out
    g = TYPES[case["grads"]]
    gates = {"none": 0, "channel": 1, "sequence": rows // case["gate_rows"]}[case["gate"]]
    out = {"df": empty(rows, cols), "dh": empty(rows, cols), "dgate": empty(gates, cols, dtype=g) if gates else None}
    for norm in ("post", "pre"):
        for p in ("gamma", "beta"):
            out[f"d{norm}_{p}"] = empty(cols, dtype=g) if case[norm] else None
    return out


# --------------------------------------------------------------------------- #
# One pass
# --------------------------------------------------------------------------- #


def run(s):
    if own:
        return _run_own(s)
    return {"act8": _plain_act8, "linear": _plain_linear, "norm_fwd": _plain_norm_fwd, "norm_bwd": _plain_norm_bwd}[s["case"]["kind"]](s)


def _run_own(s):
    case, lib, out = s["case"], s["lib"], s["out"]
    code = CODE[case["dtype"]]
    stream = torch.cuda.current_stream().cuda_stream
    p = lambda t: None if t is None else t.data_ptr()
    if case["kind"] == "act8":
        rows, cols = case["rows"], case["cols"]
        lib.mg_act8_store(p(s["x"]), p(out["act8"]), rows, cols, int(case["relu"]), code, stream)
        lib.mg_act8_load(p(out["act8"]), p(out["x"]), rows, cols, code, stream)
        return {"x": out["x"]}
    if case["kind"] == "linear":
        lib.mg_linear_bwd_act8(p(s["dy"]), p(s["x8"]), p(s["w"]), p(out["dx"]), p(out["dw"]), p(out["db"]), case["rows"],
                               case["outputs"], case["inputs"], 0, int(case["relu"]), code, CODE[case["grads"]], stream)
        return out
    if case["kind"] == "norm_fwd":
        lib.mg_residual_norm_fwd(p(s["f"]), p(s["h"]), p(s["gate"]), p(s["post_gamma"]), p(s["post_beta"]), p(s["pre_gamma"]),
                                 p(s["pre_beta"]), p(out["h_out"]), p(out["x"]), p(out["post_mean"]), p(out["post_rstd"]),
                                 p(out["pre_mean"]), p(out["pre_rstd"]), None, None, case["rows"], case["cols"],
                                 case["gate_rows"], case["scale"], EPS, code, stream)
        return out
    lib.mg_residual_norm_bwd(p(s["dx"]), p(s["dh_out"]), p(s["f"]), p(s["f8"]), p(s["h_out"]), p(s["gate"]), p(s["post_gamma"]),
                             p(s["post_beta"]), p(s["pre_gamma"]), p(s["post_mean"]), p(s["post_rstd"]), p(s["pre_mean"]),
                             p(s["pre_rstd"]), p(out["df"]), p(out["dh"]), p(out["dgate"]), p(out["dpost_gamma"]),
                             p(out["dpost_beta"]), p(out["dpre_gamma"]), p(out["dpre_beta"]), case["rows"], case["cols"],
                             case["gate_rows"], case["scale"], code, CODE[case["grads"]], stream)
    return out


def _plain_act8(s):
    case = s["case"]
    act8 = _act8_store(s["x"], case["dtype"], case["relu"])
    return {"x": _act8_load(act8, case["rows"], case["cols"]).to(TYPES[case["dtype"]])}


def _plain_linear(s):
    case = s["case"]
    t, g = TYPES[case["dtype"]], TYPES[case["grads"]]
    x = _act8_load(s["x8"], case["rows"], case["inputs"])
    dy, w = s["dy"].float(), s["w"].float()
    dx = dy @ w
    if case["relu"]:
        dx = torch.where(x > 0, dx, 0.0)
    return {"dx": dx.to(t), "dw": (dy.t() @ x).to(g), "db": dy.sum(dim=0).to(g) if case["bias"] else None}


def _plain_norm(x, gamma, beta):
    mean = x.mean(dim=1)
    centred = x - mean[:, None]
    rstd = torch.rsqrt(centred.square().mean(dim=1) + EPS)
    return centred * rstd[:, None] * gamma.float() + beta.float(), mean, rstd


def _rows_of(gate, case):
    """The gate of every row, or of all of them."""
    gate = gate.float()
    return gate if gate.shape[0] == 1 else gate.repeat_interleave(case["gate_rows"], dim=0)


def _plain_norm_fwd(s):
    case = s["case"]
    t = TYPES[case["dtype"]]
    out = {"x": None, "post_mean": None, "post_rstd": None, "pre_mean": None, "pre_rstd": None}
    z = s["f"].float()
    if case["post"]:
        z, out["post_mean"], out["post_rstd"] = _plain_norm(z, s["post_gamma"], s["post_beta"])
    if s["gate"] is not None:
        z = z * _rows_of(s["gate"], case)
    h = s["h"].float() * case["scale"] + z
    out["h_out"] = h.to(t)
    if case["pre"]:
        x, out["pre_mean"], out["pre_rstd"] = _plain_norm(h, s["pre_gamma"], s["pre_beta"])
        out["x"] = x.to(t)
    return out


def _plain_norm_grad(dy, hat, rstd):
    """What a norm passes back of dy, the gradient of its values before the affine map."""
    return rstd[:, None] * (dy - dy.mean(dim=1, keepdim=True) - hat * (dy * hat).mean(dim=1, keepdim=True))


def _plain_norm_bwd(s):
    case = s["case"]
    t, g = TYPES[case["dtype"]], TYPES[case["grads"]]
    out = {"dgate": None, "dpost_gamma": None, "dpost_beta": None, "dpre_gamma": None, "dpre_beta": None}
    d = s["dh_out"].float()
    if case["pre"]:
        dx = s["dx"].float()
        hat = (s["h_out"].float() - s["pre_mean"][:, None]) * s["pre_rstd"][:, None]
        d = d + _plain_norm_grad(dx * s["pre_gamma"].float(), hat, s["pre_rstd"])
        out["dpre_gamma"] = (dx * hat).sum(dim=0).to(g)
        out["dpre_beta"] = dx.sum(dim=0).to(g)
    out["dh"] = (d * case["scale"]).to(t)
    hat = z = s["f"].float() if s["f8"] is None else _act8_load(s["f8"], case["rows"], case["cols"])
    if case["post"]:
        hat = (z - s["post_mean"][:, None]) * s["post_rstd"][:, None]
        z = hat * s["post_gamma"].float() + s["post_beta"].float()
    u = d
    if s["gate"] is not None:
        out["dgate"] = (d * z).view(s["gate"].shape[0], -1, case["cols"]).sum(dim=1).to(g)
        u = d * _rows_of(s["gate"], case)
    if case["post"]:
        out["dpost_gamma"] = (u * hat).sum(dim=0).to(g)
        out["dpost_beta"] = u.sum(dim=0).to(g)
        u = _plain_norm_grad(u * s["post_gamma"].float(), hat, s["post_rstd"])
    out["df"] = u.to(t)
    return out


# --------------------------------------------------------------------------- #
# The same from the definitions, in 64 bits
# --------------------------------------------------------------------------- #


def exact(case, seed):
    s = _inputs(case, seed)
    return {"act8": _exact_act8, "linear": _exact_linear, "norm_fwd": _exact_norm_fwd, "norm_bwd": _exact_norm_bwd}[case["kind"]](case, s)


def _exact_power(k):
    return (k.to(torch.int64) + 1023 << 52).view(torch.float64)


def _exact_act8(case, s):
    """Block by block: the least k whose block rounds to whole numbers of at most 127."""
    x = s["x"].double()
    low, high = K_RANGE[case["dtype"]]
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], BLOCK):
        v = x[:, c:c + BLOCK]
        m = v.abs().max(dim=1, keepdim=True).values
        k = torch.ceil(torch.log2(m.clamp_min(2.0 ** -160) / 127.5))
        k = torch.where(m >= 127.5 * _exact_power(k), k + 1, k)
        k = torch.where(m < 127.5 * _exact_power(k - 1), k - 1, k)
        step = _exact_power(torch.minimum(torch.maximum(k, torch.full_like(k, low)), torch.full_like(k, high)))
        q = torch.round(v / step)
        q = torch.minimum(torch.maximum(q, torch.full_like(q, -127)), torch.full_like(q, 127))
        if case["relu"]:
            q = q + ((q == 0) & (v > 0)).double()
        out[:, c:c + BLOCK] = q * step
    return {"x": out}


def _exact_values(act8, rows, cols):
    """Values of a run of bytes: whole numbers in two's complement times powers of two."""
    ld = (cols + BLOCK - 1) // BLOCK * BLOCK
    q = act8[:rows * ld].reshape(rows, ld).double()
    q = q - 256 * (q > 127)
    step = _exact_power(act8[rows * ld:].reshape(rows, ld // BLOCK).to(torch.int64) - 133)
    return (q * step.repeat_interleave(BLOCK, dim=1))[:, :cols]


def _exact_linear(case, s):
    x = _exact_values(s["x8"], case["rows"], case["inputs"])
    dy, w = s["dy"].double(), s["w"].double()
    dx = torch.matmul(dy, w)
    if case["relu"]:
        dx *= x > 0
    db = torch.matmul(torch.ones(dy.shape[0], dtype=torch.float64, device=dy.device), dy) if case["bias"] else None
    return {"dx": dx, "dw": torch.matmul(dy.t().contiguous(), x), "db": db}


def _exact_norm_fwd(case, s):
    out = {"h_out": None, "x": None}
    f, h = s["f"].double(), s["h"].double()

    def stats(v, name):
        mean = v.sum(dim=1) / v.shape[1]
        var = (v * v).sum(dim=1) / v.shape[1] - mean * mean
        out[name + "_mean"], out[name + "_rstd"] = mean, 1 / torch.sqrt(var + EPS)
        return (v - mean.unsqueeze(1)) / torch.sqrt(var + EPS).unsqueeze(1)

    for name in ("post", "pre"):
        out[name + "_mean"] = out[name + "_rstd"] = None
    if case["post"]:
        f = stats(f, "post") * s["post_gamma"].double() + s["post_beta"].double()
    if s["gate"] is not None:
        at = torch.arange(case["rows"], device=f.device) // case["gate_rows"]
        f = f * s["gate"].double()[at]
    out["h_out"] = case["scale"] * h + f
    if case["pre"]:
        out["x"] = stats(out["h_out"], "pre") * s["pre_gamma"].double() + s["pre_beta"].double()
    return out


def _exact_norm_bwd(case, s):
    """By the chain rule over rows, and with sums over rows as products with a vector of ones."""
    D = lambda name: None if s[name] is None else s[name].double()
    rows, cols = case["rows"], case["cols"]
    ones = torch.ones(rows, dtype=torch.float64, device="cuda")
    column_sums = lambda v: torch.matmul(ones, v)
    out = {"dgate": None, "dpost_gamma": None, "dpost_beta": None, "dpre_gamma": None, "dpre_beta": None}
    total = D("dh_out")
    if case["pre"]:
        r = D("pre_rstd").unsqueeze(1)
        n = (D("h_out") - D("pre_mean").unsqueeze(1)) * r
        dn = D("dx") * D("pre_gamma")
        total = total + r * dn - r * dn.sum(dim=1, keepdim=True) / cols - r * n * (dn * n).sum(dim=1, keepdim=True) / cols
        out["dpre_gamma"], out["dpre_beta"] = column_sums(D("dx") * n), column_sums(D("dx"))
    out["dh"] = case["scale"] * total
    f = _exact_values(s["f8"], rows, cols) if s["f"] is None else D("f")
    gate = 1.0
    if s["gate"] is not None:
        at = torch.arange(rows, device="cuda") // case["gate_rows"]
        gate = D("gate")[at]
    if case["post"]:
        r = D("post_rstd").unsqueeze(1)
        n = (f - D("post_mean").unsqueeze(1)) * r
        z = n * D("post_gamma") + D("post_beta")
    else:
        z = f
    if s["gate"] is not None:
        out["dgate"] = torch.zeros(s["gate"].shape, dtype=torch.float64, device="cuda").index_add_(0, at, total * z)
    dz = total * gate
    if case["post"]:
        out["dpost_gamma"], out["dpost_beta"] = column_sums(dz * n), column_sums(dz)
        dn = dz * D("post_gamma")
        dz = r * dn - r * dn.sum(dim=1, keepdim=True) / cols - r * n * (dn * n).sum(dim=1, keepdim=True) / cols
    out["df"] = dz
    return out
