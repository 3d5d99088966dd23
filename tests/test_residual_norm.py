"""The residual path between two blocks (norm, gate, scaled residual sum, norm) against float64, forward and backward.

Tolerances, per value: half a step of the output's type, plus fp32 rounding, 2^-24 of the magnitudes that the formula adds up
(the same formula with absolute values everywhere) for each of the at most 64 roundings that lie on the way of a value through
a row (16 additions in a thread, 6 steps over lanes, 16 waves, and the arithmetic of the two norms), or, for sums over rows,
through the additions of a column: 64 and the rows that one thread adds.
"""
import ctypes as C

import numpy as np
import pytest

from helpers import normal
from oracle import oracle_np as O

import mograd_amd
from mograd_amd import BF16, F16, F32, I32, I64, AnyBuffer, MogradError
from mograd_amd.runtime import round_to_dtype

KIND = {F32: "f32", F16: "f16", BF16: "bf16"}
EPS = {F32: 2.0 ** -23, F16: 2.0 ** -10, BF16: 2.0 ** -7}
FLOATS = [F32, F16, BF16]
U = 2.0 ** -24
LN_EPS = 1e-5


# ---- the oracle, no GPU --------------------------------------------------------------------


@pytest.mark.parametrize("gates", [0, 1, 3])
@pytest.mark.parametrize("post,pre", [(1, 1), (0, 1), (1, 0), (0, 0)])
def test_oracle_gradients(gates, post, pre):
    """The formulas against central differences of the forward's and against autograd."""
    import torch

    rng = np.random.default_rng(5)
    rows, cols, scale = 12, 9, 0.75
    p = {"f": rng.standard_normal((rows, cols)), "h": rng.standard_normal((rows, cols)) * 2 + 1}
    if gates:
        p["gate"] = rng.standard_normal((gates, cols))
    for name, on in (("post", post), ("pre", pre)):
        if on:
            p[name + "_gamma"], p[name + "_beta"] = rng.standard_normal(cols), rng.standard_normal(cols)
    dx, dh_out = rng.standard_normal((rows, cols)), rng.standard_normal((rows, cols))

    def forward(q):
        return O.residual_norm_fwd(q["f"], q["h"], q.get("gate"), (q["post_gamma"], q["post_beta"]) if post else None,
                                   (q["pre_gamma"], q["pre_beta"]) if pre else None, scale, LN_EPS)

    def objective(q):
        out = forward(q)
        return (out["h_out"] * dh_out).sum() + ((out["x"] * dx).sum() if pre else 0)

    out = forward(p)
    got = O.residual_norm_bwd(dx if pre else None, dh_out, p["f"], out["h_out"], p.get("gate"),
                              (p["post_gamma"], p["post_beta"], out["post_mean"], out["post_rstd"]) if post else None,
                              (p["pre_gamma"], p["pre_beta"], out["pre_mean"], out["pre_rstd"]) if pre else None, scale)
    t = {k: torch.tensor(v, requires_grad=True) for k, v in p.items()}
    z = t["f"]
    if post:
        z = torch.nn.functional.layer_norm(z, (cols,), t["post_gamma"], t["post_beta"], LN_EPS)
    if gates:
        z = z * t["gate"].repeat_interleave(rows // gates, 0)
    h = scale * t["h"] + z
    total = (h * torch.tensor(dh_out)).sum()
    if pre:
        total = total + (torch.nn.functional.layer_norm(h, (cols,), t["pre_gamma"], t["pre_beta"], LN_EPS) * torch.tensor(dx)).sum()
    total.backward()
    for name, value in p.items():
        grad = got["d" + name]
        np.testing.assert_allclose(grad, t[name].grad.numpy(), rtol=1e-9, atol=1e-10)
        flat = value.reshape(-1)
        for i in rng.integers(0, flat.size, 3):
            step = 1e-6
            keep = flat[i]
            flat[i] = keep + step
            up = objective(p)
            flat[i] = keep - step
            down = objective(p)
            flat[i] = keep
            np.testing.assert_allclose((up - down) / (2 * step), grad.reshape(-1)[i], rtol=1e-5, atol=1e-6)


def test_refusals():
    """Answered before anything is launched; the pointers are never followed."""
    lib = mograd_amd.load()
    p, odd = C.c_void_p(4096), C.c_void_p(4100)

    def fwd(f=p, h=p, gate=p, post=(p, p, p, p), pre=(p, p, p, p), h_out=p, x=p, f8=None, x8=None, rows=8, cols=4, gate_rows=4, dtype=F32):
        return lib.mg_residual_norm_fwd(f, h, gate, post[0], post[1], pre[0], pre[1], h_out, x, post[2], post[3], pre[2], pre[3],
                                        f8, x8, rows, cols, gate_rows, 1.0, 1e-5, dtype, None)

    def bwd(dx=p, dh_out=p, f=p, f8=None, h_out=p, gate=p, post=(p, p, p, p), pre=(p, p, p), df=p, dh=p, dgate=p, dpost=(p, p),
            dpre=(p, p), rows=8, cols=4, gate_rows=4, dtype=F32, grads=F32):
        return lib.mg_residual_norm_bwd(dx, dh_out, f, f8, h_out, gate, *post[:2], pre[0], *post[2:], *pre[1:], df, dh, dgate,
                                        *dpost, *dpre, rows, cols, gate_rows, 1.0, dtype, grads, None)

    none4, some = (None,) * 4, (p, None, p, p)
    common = [dict(dtype=I32), dict(dtype=7), dict(rows=-1), dict(cols=0), dict(cols=1 << 30), dict(rows=1 << 31, gate_rows=1),
              dict(gate_rows=3), dict(gate_rows=0), dict(gate_rows=-4), dict(gate_rows=16), dict(f=None), dict(post=some)]
    for bad in common + [dict(h=None), dict(h_out=None), dict(pre=some), dict(x=None), dict(pre=none4), dict(f8=odd), dict(x8=odd),
                         dict(pre=none4, x=None, x8=p)]:
        with pytest.raises(MogradError) as e:
            fwd(**bad)
        assert e.value.status == 1 and "residual_norm_fwd" in str(e.value), bad
    for bad in common + [dict(dtype=F16, grads=BF16), dict(grads=I64), dict(dgate=None), dict(gate=None), dict(f8=p), dict(f=None, f8=odd),
                         dict(f=None, post=none4, dpost=(None, None)), dict(df=None), dict(dh=None), dict(h_out=None), dict(dpost=(p, None)), dict(dpre=(None, p)), dict(dx=None),
                         dict(post=none4), dict(pre=(None,) * 3, dx=None, dpre=(None, None), dh_out=None)]:
        with pytest.raises(MogradError) as e:
            bwd(**bad)
        assert e.value.status == 1 and "residual_norm_bwd" in str(e.value), bad
    assert fwd(rows=0) == 0


# ---- on the GPU ----------------------------------------------------------------------------


class _Place:
    """Device copies of arrays, each starting `offset` elements into its buffer, with guards on both sides of what is written."""

    def __init__(self, device, offset):
        self.device, self.offset, self.out = device, offset, {}

    def put(self, a, dtype):
        if a is None:
            return None
        a = np.asarray(a, np.float32).reshape(-1)
        buf = AnyBuffer.from_numpy(self.device, np.concatenate([np.full(self.offset, -3.0, np.float32), a, np.full(9, -3.0, np.float32)]), dtype)
        self.out[id(buf)] = buf  # keeps it
        return AnyBuffer(buf.storage, dtype, a.size, self.offset)

    def new(self, name, shape, dtype):
        b = self.put(np.full(shape, 77.0), dtype)
        self.out[name] = (b, shape)
        return b

    def read(self, name):
        b, shape = self.out[name]
        whole = AnyBuffer(b.storage, b.dtype, self.offset + b.numel + 9, 0).to_numpy()
        assert (whole[:self.offset] == -3).all() and (whole[self.offset + b.numel:] == -3).all(), f"{name}: written outside"
        return whole[self.offset:self.offset + b.numel].reshape(shape)


def _ptr(b):
    return None if b is None else b.data_ptr()


def _upload_bytes(device, data):
    padded = np.zeros(-(-len(data) // 4) * 4, np.uint8)
    padded[:len(data)] = data
    return AnyBuffer.from_numpy(device, padded.view(np.int32), I32)


def _inputs(seed, rows, cols, gates, post, pre, dtype):
    r = lambda i, shape, std=1.0, mean=0.0: round_to_dtype(normal(seed, i, shape, std, mean), dtype)
    size = np.exp(0.5 * normal(seed, 20, (1, cols)))
    p = {"f": round_to_dtype(normal(seed, 0, (rows, cols)) * size, dtype), "h": r(1, (rows, cols), 2.0, 0.5)}
    p["gate"] = r(2, (gates, cols), 0.3, 0.5) if gates else None
    p["post"] = (r(3, cols, 0.25, 1.0), r(4, cols, 0.1)) if post else None
    p["pre"] = (r(5, cols, 0.25, 1.0), r(6, cols, 0.1)) if pre else None
    p["dx"] = r(7, (rows, cols), 0.05) if pre else None
    p["dh_out"] = r(8, (rows, cols), 0.05)
    return p


def _forward(device, p, dtype, scale, offset=0, in_place=False, keep8=False):
    rows, cols = p["f"].shape
    place = _Place(device, offset)
    gates = 0 if p["gate"] is None else len(p["gate"])
    f, h, gate = (place.put(p[k], dtype) for k in ("f", "h", "gate"))
    post = [place.put(a, dtype) for a in p["post"] or (None, None)]
    pre = [place.put(a, dtype) for a in p["pre"] or (None, None)]
    if in_place:
        h_out = h
        place.out["h_out"] = (h, (rows, cols))
    else:
        h_out = place.new("h_out", (rows, cols), dtype)
    x = place.new("x", (rows, cols), dtype) if p["pre"] else None
    stats = {n: place.new(n, (rows,), F32) if p[n.split("_")[0]] else None for n in ("post_mean", "post_rstd", "pre_mean", "pre_rstd")}
    n8 = device.lib.mg_act8_bytes(rows, cols)
    f8, x8 = (AnyBuffer.create(I32, device, -(-n8 // 4) + 1, fill=0x55) if keep else None for keep in (keep8, keep8 and p["pre"]))
    device.lib.mg_residual_norm_fwd(_ptr(f), _ptr(h), _ptr(gate), *map(_ptr, post), *map(_ptr, pre), _ptr(h_out), _ptr(x),
                                    *map(_ptr, stats.values()), _ptr(f8), _ptr(x8), rows, cols, rows // gates if gates else 0, scale,
                                    LN_EPS, dtype, device.stream)
    out = {"h_out": place.read("h_out"), "x": place.read("x") if x else None}
    for n, b in stats.items():
        out[n] = place.read(n) if b else None
    for n, b in (("f8", f8), ("x8", x8)):
        out[n] = b.to_numpy().view(np.uint8)[:n8] if b else None
    return out


def _close(got, want, bound, what):
    assert got.shape == want.shape, what
    assert np.isfinite(got).all(), what
    ratio = np.abs(got - want) / np.maximum(bound, 1e-300)
    if got.size and ratio.max() > 1:
        at = np.unravel_index(ratio.argmax(), ratio.shape)
        pytest.fail(f"{what}{list(map(int, at))}: {got[at]!r}, not {want[at]!r}: {ratio[at]:.3g} of the bound")


def _half_step(want, dtype):
    """What one rounding to the type may change: half of eps relative to the value, and never less than half of the spacing that
    fp16 has below 2^-14, 2^-24 (fp32 and bf16 go on to 2^-126)."""
    return np.maximum(EPS[dtype] / 2 * np.abs(want), 2.0 ** -25 if dtype == F16 else 0.0)


def _row_max(a):
    return np.abs(a).max(axis=1, keepdims=True)


def _check_forward(p, got, dtype, scale):
    want = O.residual_norm_fwd(p["f"], p["h"], p["gate"], p["post"], p["pre"], scale, LN_EPS)
    rows = len(p["f"])
    z = np.abs(p["f"]).astype(np.float64)
    gate = np.repeat(np.abs(p["gate"]), rows // len(p["gate"]), axis=0) if p["gate"] is not None else 1.0
    if p["post"]:  # the mean's error is that of a sum of the row's magnitudes
        rstd = want["post_rstd"][:, None]
        _close(got["post_mean"], want["post_mean"], 64 * U * _row_max(p["f"])[:, 0], "post_mean")
        # of the variance: relative, and of the mean's square where the mean is what the values have in common
        spread = 64 * U * (1 + (_row_max(p["f"]) * rstd) ** 2 * 64 * U)
        _close(got["post_rstd"], want["post_rstd"], (rstd * spread)[:, 0], "post_rstd")
        z = _row_max(p["f"]) * rstd * np.abs(p["post"][0]) + np.abs(p["post"][1])
    mag = np.abs(scale * p["h"]) + gate * z
    _close(got["h_out"], want["h_out"], _half_step(want["h_out"], dtype) + 64 * U * mag, "h_out")
    if p["pre"]:
        rstd = want["pre_rstd"][:, None]
        _close(got["pre_mean"], want["pre_mean"], 128 * U * _row_max(mag)[:, 0], "pre_mean")
        _close(got["pre_rstd"], want["pre_rstd"], (rstd * 128 * U * (1 + _row_max(mag) * rstd))[:, 0], "pre_rstd")
        bound = 128 * U * ((1 + _row_max(mag) * rstd) ** 2 * np.abs(p["pre"][0]) + np.abs(p["pre"][1]))
        _close(got["x"], want["x"], _half_step(want["x"], dtype) + bound, "x")


def _check_kept(p, got, dtype):
    """f8 and x8: what storing f and x gives."""
    assert np.array_equal(got["f8"], O.act8_store(p["f"], KIND[dtype]))
    if p["pre"]:
        assert np.array_equal(got["x8"], O.act8_store(got["x"], KIND[dtype]))


def _backward(device, p, saved, dtype, grads, scale, offset=0, in_place=False, act8=False, skip=False, shape=None):
    rows, cols = shape or p["f"].shape
    place = _Place(device, offset)
    gates = 0 if p["gate"] is None else len(p["gate"])
    put = lambda a, t=dtype: place.put(a, t)
    post = [put(a) for a in p["post"] or (None, None)]
    pre_gamma = put(p["pre"][0]) if p["pre"] else None
    stats = [put(saved[n], F32) for n in ("post_mean", "post_rstd", "pre_mean", "pre_rstd")]
    dx, dh_out, gate = put(p["dx"]), None if skip else put(p["dh_out"]), put(p["gate"])
    h_out = put(saved["h_out"]) if p["pre"] else None
    f8 = _upload_bytes(device, O.act8_store(p["f"], KIND[dtype])) if act8 else None
    f = None if act8 else put(p["f"])
    df = place.new("df", (rows, cols), dtype)
    if in_place:
        dh = dh_out
        place.out["dh"] = (dh_out, (rows, cols))
    else:
        dh = place.new("dh", (rows, cols), dtype)
    new = lambda n, shape, on: place.new(n, shape, grads) if on else None
    outs = [new("dgate", (gates, cols), gates), new("dpost_gamma", (cols,), p["post"]), new("dpost_beta", (cols,), p["post"]),
            new("dpre_gamma", (cols,), p["pre"]), new("dpre_beta", (cols,), p["pre"])]
    device.lib.mg_residual_norm_bwd(_ptr(dx), _ptr(dh_out), _ptr(f), _ptr(f8), _ptr(h_out), _ptr(gate), *map(_ptr, post), _ptr(pre_gamma),
                                    *map(_ptr, stats), _ptr(df), _ptr(dh), *map(_ptr, outs), rows, cols, rows // gates if gates else 0,
                                    scale, dtype, grads, device.stream)
    return {n: place.read(n) for n in ("df", "dh", "dgate", "dpost_gamma", "dpost_beta", "dpre_gamma", "dpre_beta") if n in place.out}


def _saved(p, dtype, scale):
    """What a forward pass leaves: h_out rounded, statistics in fp32."""
    out = O.residual_norm_fwd(p["f"], p["h"], p["gate"], p["post"], p["pre"], scale, LN_EPS)
    saved = {"h_out": round_to_dtype(out["h_out"], dtype)}
    for n in ("post_mean", "post_rstd", "pre_mean", "pre_rstd"):
        saved[n] = None if out[n] is None else out[n].astype(np.float32)
    return saved


def _check_backward(p, saved, got, dtype, grads, scale, act8=False, skip=False):
    rows, cols = p["f"].shape
    f = O.act8_load(O.act8_store(p["f"], KIND[dtype]), rows, cols) if act8 else p["f"].astype(np.float64)
    dh_out = None if skip else p["dh_out"]
    post = (*p["post"], saved["post_mean"], saved["post_rstd"]) if p["post"] else None
    pre = (*p["pre"], saved["pre_mean"], saved["pre_rstd"]) if p["pre"] else None
    want = O.residual_norm_bwd(p["dx"], dh_out, f, saved["h_out"], p["gate"], post, pre, scale)
    # the same formulas over magnitudes
    d = np.zeros((rows, cols)) if skip else np.abs(p["dh_out"]).astype(np.float64)
    sums = {}
    if pre:
        rstd = saved["pre_rstd"][:, None].astype(np.float64)
        hat = (np.abs(saved["h_out"]) + np.abs(saved["pre_mean"])[:, None]) * rstd
        dg = np.abs(p["dx"] * p["pre"][0])
        d = d + rstd * (dg + dg.mean(1, keepdims=True) + hat * (dg * hat).mean(1, keepdims=True))
        sums["dpre_gamma"], sums["dpre_beta"] = np.abs(p["dx"]) * hat, np.abs(p["dx"])
    mag = {"dh": np.abs(scale) * d}
    gate = np.repeat(np.abs(p["gate"]), rows // len(p["gate"]), axis=0) if p["gate"] is not None else 1.0
    u, hat = d * gate, np.abs(f)
    if post:
        rstd = saved["post_rstd"][:, None].astype(np.float64)
        hat = (np.abs(f) + np.abs(saved["post_mean"])[:, None]) * rstd
        sums["dpost_gamma"], sums["dpost_beta"] = u * hat, u
        ug = u * np.abs(p["post"][0])
        u = rstd * (ug + ug.mean(1, keepdims=True) + hat * (ug * hat).mean(1, keepdims=True))
    mag["df"] = u
    for n in ("dh", "df"):
        _close(got[n], want[n], _half_step(want[n], dtype) + 64 * U * mag[n], n)
    # (a column's parts: 64 roundings for each value before it is added, and the additions of at most rows / 16 + 64 of them)
    chain = 128 + rows / 16
    for n, terms in sums.items():
        _close(got[n], want[n], _half_step(want[n], grads) + chain * U * terms.sum(0), n)
    if p["gate"] is not None:
        z = hat * np.abs(p["post"][0]) + np.abs(p["post"][1]) if post else hat
        terms = (d * z).reshape(len(p["gate"]), -1, cols).sum(1)
        _close(got["dgate"], want["dgate"], _half_step(want["dgate"], grads) + chain * U * terms, "dgate")


# rows, cols, gates: fewer columns than a chunk, one row, odd widths, every row layout (16 lanes to 1024 threads), rows that
# registers do not hold, one gate row to one for every row
SHAPES = [(1, 1, 1), (6, 3, 2), (1, 8, 0), (5, 33, 5), (130, 64, 1), (130, 64, 13), (67, 130, 1), (96, 256, 3), (40, 384, 4), (33, 500, 0),
          (24, 1001, 3), (9, 2056, 1), (10, 4096, 2), (6, 4100, 0), (4, 8200, 2), (3, 16384, 1), (3, 20001, 3), (2, 70000, 1),
          (3001, 96, 1), (2600, 40, 1300), (1500, 200, 5)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,cols,gates", SHAPES)
@pytest.mark.parametrize("post,pre", [(1, 1), (0, 1), (1, 0), (0, 0)])
def test_forward(device, rows, cols, gates, post, pre, dtype):
    p = _inputs(31, rows, cols, gates, post, pre, dtype)
    got = _forward(device, p, dtype, 0.75, keep8=True)
    _check_forward(p, got, dtype, 0.75)
    _check_kept(p, got, dtype)
    off = _forward(device, p, dtype, 0.75, offset=1, in_place=True)
    _check_forward(p, off, dtype, 0.75)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,grads", [(F32, F32), (F16, F16), (BF16, F32)])
@pytest.mark.parametrize("rows,cols,gates", SHAPES)
@pytest.mark.parametrize("post,pre", [(1, 1), (0, 1), (1, 0), (0, 0)])
def test_backward(device, rows, cols, gates, post, pre, dtype, grads):
    p = _inputs(32, rows, cols, gates, post, pre, dtype)
    saved = _saved(p, dtype, 1.25)
    for kw, run in ((dict(), dict()), (dict(), dict(offset=1, in_place=True)), (dict(act8=True), dict()),
                    (dict(act8=True, skip=bool(pre)), dict(offset=1))):
        got = _backward(device, p, saved, dtype, grads, 1.25, **kw, **run)
        _check_backward(p, saved, got, dtype, grads, 1.25, **kw)


# rows, cols, gates: more gate rows than workgroups, and than rows in flight at once, of every layout
MANY_GATES = [(9100, 40, 4550), (4400, 200, 2200), (2400, 500, 1200), (2210, 1001, 1105), (1600, 384, 400), (700, 130, 350), (300, 4096, 300),
              (2100, 3, 2100), (520, 8200, 260)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,grads", [(F32, F32), (F16, F16), (BF16, F32)])
@pytest.mark.parametrize("rows,cols,gates", MANY_GATES)
@pytest.mark.parametrize("post,pre", [(1, 1), (0, 1), (1, 0)])
def test_backward_of_many_gate_rows(device, rows, cols, gates, post, pre, dtype, grads):
    p = _inputs(36, rows, cols, gates, post, pre, dtype)
    saved = _saved(p, dtype, 1.25)
    for kw, run in ((dict(), dict()), (dict(act8=True), dict(offset=1))):
        got = _backward(device, p, saved, dtype, grads, 1.25, **kw, **run)
        _check_backward(p, saved, got, dtype, grads, 1.25, **kw)
        again = _backward(device, p, saved, dtype, grads, 1.25, **kw, **run)
        assert all(np.array_equal(got[n], again[n]) for n in got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
def test_first_column_far_from_the_others(device, dtype):
    """A column a thousand times the others, at the place that a shifted sum would take for its shift, and a large common mean."""
    p = _inputs(33, 50, 384, 1, 1, 1, dtype)
    p["f"][:, 0] = round_to_dtype(p["f"][:, 0] * 1000 + 500, dtype)
    p["h"][25:] = round_to_dtype(p["h"][25:] + 100, dtype)
    _check_forward(p, _forward(device, p, dtype, 1.0), dtype, 1.0)
    saved = _saved(p, dtype, 1.0)
    _check_backward(p, saved, _backward(device, p, saved, dtype, F32, 1.0), dtype, F32, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("cols", [64, 100, 384, 4096])
def test_rows_do_not_touch_each_other(device, dtype, cols):
    """A NaN and an infinity in one row stay in that row; rows of one value have zero spread and no division by zero."""
    p = _inputs(34, 21, cols, 1, 1, 1, dtype)
    clean = _forward(device, p, dtype, 1.0)
    p["f"][4, cols // 2] = np.nan
    p["h"][9, cols - 1] = np.inf
    p["f"][12] = 2.5
    p["h"][13], p["f"][13] = 0, 0
    got = _forward(device, p, dtype, 1.0)
    same = [r for r in range(21) if r not in (4, 9, 12, 13)]
    for n in ("h_out", "x", "post_mean", "post_rstd", "pre_mean", "pre_rstd"):
        assert np.array_equal(got[n][same], clean[n][same]), n
    assert np.isnan(got["x"][4]).all() and np.isnan(got["x"][9]).all()
    assert np.isfinite(got["x"][12:14]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [33, 384, 70000])
def test_backward_without_f(device, cols):
    """Neither a gate nor a post norm: f is not asked for."""
    p = _inputs(37, 12, cols, 0, 0, 1, F32)
    saved = _saved(p, F32, 0.5)
    want = _backward(device, p, saved, F32, F32, 0.5)
    _check_backward(p, saved, want, F32, F32, 0.5)
    got = _backward(device, dict(p, f=None), saved, F32, F32, 0.5, shape=(12, cols))
    for n in want:
        assert np.array_equal(got[n], want[n]), n


@pytest.mark.gpu
def test_twice_gives_the_same_bits(device):
    p = _inputs(35, 4000, 256, 8, 1, 1, BF16)
    saved = _saved(p, BF16, 1.0)
    a, b = (_backward(device, p, saved, BF16, F32, 1.0) for _ in range(2))
    for n in a:
        assert np.array_equal(a[n], b[n]), n


@pytest.mark.gpu
def test_no_rows(device):
    p = {n: AnyBuffer.create(F32, device, 8, fill=3.0) for n in ("gate", "dgate", "dg", "db", "pg", "pb")}
    q = {n: _ptr(b) for n, b in p.items()}
    one = q["gate"]
    device.lib.mg_residual_norm_bwd(one, one, one, None, one, q["gate"], one, one, one, one, one, one, one, one, one, q["dgate"], q["dg"],
                                    q["db"], q["pg"], q["pb"], 0, 8, 0, 1.0, F32, F32, device.stream)
    for n in ("dgate", "dg", "db", "pg", "pb"):
        assert (p[n].to_numpy() == 0).all(), n
    assert (p["gate"].to_numpy() == 3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,cols", [(300, 384), (77, 1001)])
def test_forward_then_backward(device, dtype, rows, cols):
    """The two as they are used together: the forward keeps f in 8 bits, the backward reads that and the forward's statistics."""
    p = _inputs(36, rows, cols, 1, 1, 1, dtype)
    out = _forward(device, p, dtype, 1.0, keep8=True)
    got = _backward(device, p, out, dtype, F32, 1.0, act8=True)
    _check_backward(p, out, got, dtype, F32, 1.0, act8=True)
