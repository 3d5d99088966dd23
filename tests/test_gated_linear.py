"""Gated Linear layers against float64, forward and backward.

Tolerances, per value.  A product's fp32 sum of K terms is off by at most (K + 16) 2^-24 of the sum of its terms' magnitudes (a rounding
a term at the worst, and the bias).  act and act' are off by the error of the projection times their largest slopes (1.2 for act, 1 for
act'), and by 2^-24 (32 + 8 g^2) of their own magnitudes (that of g u where they cross zero): a few units in the last place, and what the
rounded argument of an exponential of up to g^2 / 2 (or 1.6 g + 0.072 g^3) changes.  Each output, and the gradients of the projections
that the products take, is rounded once: half a step.
"""
import ctypes as C

import numpy as np
import pytest

from helpers import normal
from oracle import oracle_np as O
from test_residual_norm import EPS, FLOATS, U, _Place, _close, _half_step, _ptr

import mograd_amd
from mograd_amd import BF16, F16, F32, I32, I64, AnyBuffer, MogradError
from mograd_amd.runtime import round_to_dtype

GATES = O.GATES


def test_oracle_gradients():
    """The formulas against differences and autograd."""
    import torch

    rng = np.random.default_rng(1)
    M, F, K = 5, 4, 3
    x, w, b, dy = (rng.standard_normal(s) for s in ((M, K), (2 * F, K), 2 * F, (M, F)))
    acts = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "sigmoid": torch.sigmoid, "relu": torch.relu,
            "gelu_tanh": lambda g: torch.nn.functional.gelu(g, approximate="tanh")}
    for gate in GATES:
        y, gu = O.gated_linear_fwd(x, w, b, gate)
        dx, dw, db, _ = O.gated_linear_bwd(dy, gu, x, w, gate)
        t = [torch.tensor(a, requires_grad=True) for a in (x, w, b)]
        p = torch.nn.functional.linear(t[0], t[1], t[2])
        out = acts[gate](p[:, :F]) * p[:, F:]
        np.testing.assert_allclose(y, out.detach().numpy(), rtol=1e-12, atol=1e-13)
        (out * torch.tensor(dy)).sum().backward()
        for got, v in zip((dx, dw, db), t):
            np.testing.assert_allclose(got, v.grad.numpy(), rtol=1e-10, atol=1e-12)
        step = 1e-6
        for i in range(K):
            up, down = x.copy(), x.copy()
            up[1, i] += step
            down[1, i] -= step
            slope = ((O.gated_linear_fwd(up, w, b, gate)[0] - O.gated_linear_fwd(down, w, b, gate)[0]) * dy).sum() / (2 * step)
            np.testing.assert_allclose(slope, dx[1, i], rtol=1e-6, atol=1e-8)


def test_refusals():
    """Answered before anything is launched; the pointers are never followed."""
    lib = mograd_amd.load()
    p = C.c_void_p(4096)

    def fwd(x=p, w=p, bias=None, y=p, gu=None, M=4, F=8, K=8, gate=0, dtype=BF16):
        return lib.mg_gated_linear_fwd(x, w, bias, y, gu, M, F, K, gate, dtype, None)

    def bwd(dy=p, gu=p, x=p, w=p, dx=p, dw=p, db=None, M=4, F=8, K=8, gate=0, dtype=BF16, grads=BF16, deferred=False, pending=p):
        if deferred:
            return lib.mg_gated_linear_bwd_deferred(dy, gu, x, w, dx, dw, db, M, F, K, 0, gate, dtype, grads, pending, None)
        return lib.mg_gated_linear_bwd(dy, gu, x, w, dx, dw, db, M, F, K, 0, gate, dtype, grads, None)

    common = [dict(dtype=I32), dict(dtype=9), dict(gate=-1), dict(gate=5), dict(M=-1), dict(F=0), dict(K=0), dict(M=1 << 31), dict(F=1 << 30),
              dict(K=1 << 31), dict(x=None), dict(w=None)]
    for bad in common + [dict(y=None)]:
        with pytest.raises(MogradError) as e:
            fwd(**bad)
        assert e.value.status == 1 and "gated_linear_fwd" in str(e.value), bad
    for bad in common + [dict(dy=None), dict(gu=None), dict(dw=None), dict(grads=I64), dict(grads=F16), dict(dtype=F32, grads=BF16)]:
        for kw in (dict(), dict(deferred=True)):
            with pytest.raises(MogradError) as e:
                bwd(**bad, **kw)
            assert e.value.status == 1 and "gated_linear_bwd" in str(e.value), bad
    with pytest.raises(MogradError) as e:
        bwd(deferred=True, pending=None)
    assert e.value.status == 1
    for call in (fwd, bwd):
        with pytest.raises(MogradError) as e:
            call(K=1 << 22)
        assert e.value.status == 2
    assert fwd(M=0, x=None, w=None, y=None) == 0


# ---- on the GPU ----------------------------------------------------------------------------


def _inputs(seed, M, F, K, dtype, bias=True):
    r = lambda i, shape, std=1.0: round_to_dtype(normal(seed, i, shape, std), dtype)
    p = {"x": round_to_dtype(normal(seed, 0, (M, K)) * np.exp(0.5 * normal(seed, 9, (1, K))), dtype), "w": r(1, (2 * F, K), 1.4 * (1.3 * K) ** -0.5),
         "bias": r(2, 2 * F, 0.3) if bias else None, "dy": r(3, (M, F), 0.5), "gu": r(4, (M, 2 * F), 1.5)}
    return p


def _act_error(g, gate, dg):
    """How far act(g) and act'(g) may be off, from g that is off by dg."""
    act, slope = O.gate_act(g, gate)
    rel = U * (32 + 8 * np.minimum(g * g, 200.0))
    return 1.2 * dg + rel * (np.abs(act) + U), dg + rel * (np.abs(slope) + np.abs(g) + 1)


def _forward(device, p, dtype, gate, keep=True, offset=0):
    (M, K), F = p["x"].shape, len(p["w"]) // 2
    place = _Place(device, offset)
    x, w, bias = (place.put(p[k], dtype) for k in ("x", "w", "bias"))
    y, gu = place.new("y", (M, F), dtype), place.new("gu", (M, 2 * F), dtype) if keep else None
    device.lib.mg_gated_linear_fwd(_ptr(x), _ptr(w), _ptr(bias), _ptr(y), _ptr(gu), M, F, K, GATES.index(gate), dtype, device.stream)
    return place.read("y"), place.read("gu") if keep else None


def _check_forward(p, got, dtype, gate):
    y, gu = got
    want_y, want = O.gated_linear_fwd(p["x"], p["w"], p["bias"], gate)
    F, K = len(p["w"]) // 2, p["x"].shape[1]
    mass = np.abs(p["x"]).astype(np.float64) @ np.abs(p["w"]).astype(np.float64).T + (0 if p["bias"] is None else np.abs(p["bias"]))
    off = (K + 16) * U * mass
    if gu is not None:
        _close(gu, want, _half_step(want, dtype) + off, "gu")
    act = np.abs(O.gate_act(want[:, :F], gate)[0])
    act_off, _ = _act_error(want[:, :F], gate, off[:, :F])
    u = np.abs(want[:, F:]) + off[:, F:]
    _close(y, want_y, _half_step(want_y, dtype) + act_off * u + act * off[:, F:] + 4 * U * act * u, "y")


def _backward(device, p, dtype, grads, gate, offset=0, accumulate=None, dx=True, db=True, pending=None):
    (M, K), F = p["x"].shape, len(p["w"]) // 2
    place = _Place(device, offset)
    dy, gu, x, w = (place.put(p[k], dtype) for k in ("dy", "gu", "x", "w"))
    out_dx = out_db = None
    if accumulate is not None:
        out_dx = place.put(accumulate, dtype)
        place.out["dx"] = (out_dx, (M, K))
    elif dx:
        out_dx = place.new("dx", (M, K), dtype)
    out_dw = place.new("dw", (2 * F, K), grads)
    if db:
        out_db = place.new("db", (2 * F,), grads)
    args = (_ptr(dy), _ptr(gu), _ptr(x), _ptr(w) if dx else None, _ptr(out_dx), _ptr(out_dw), _ptr(out_db), M, F, K, int(accumulate is not None),
            GATES.index(gate), dtype, grads)
    if pending is None:
        device.lib.mg_gated_linear_bwd(*args, device.stream)
    else:
        device.lib.mg_gated_linear_bwd_deferred(*args, pending, device.stream)
        device.lib.mg_finish_deferred(pending, device.stream)
    return {n: place.read(n) for n in ("dx", "dw", "db") if n in place.out}


def _check_backward(p, got, dtype, grads, gate, accumulate=None):
    dx, dw, db, d = O.gated_linear_bwd(p["dy"], p["gu"], p["x"], p["w"], gate)
    (M, K), F = p["x"].shape, len(p["w"]) // 2
    g, u, dy = np.abs(p["gu"][:, :F]).astype(np.float64), np.abs(p["gu"][:, F:]), np.abs(p["dy"])
    act_off, slope_off = _act_error(p["gu"][:, :F].astype(np.float64), gate, 0.0)
    off = np.concatenate([dy * u * slope_off, dy * act_off], axis=1) + 4 * U * np.abs(d)
    off = off + _half_step(np.abs(d) + off, dtype)
    mag, w, x = np.abs(d) + off, np.abs(p["w"]).astype(np.float64), np.abs(p["x"]).astype(np.float64)
    bounds = {"dx": off @ w + (2 * F + 16) * U * (mag @ w), "dw": off.T @ x + (M + 16) * U * (mag.T @ x), "db": off.sum(0) + (M + 16) * U * mag.sum(0)}
    want = {"dx": dx, "dw": dw, "db": db}
    if accumulate is not None and "dx" in got:
        # 16 bits: the product is rounded before it is added, the sum after
        bounds["dx"] = bounds["dx"] + _half_step(np.abs(dx) + bounds["dx"], dtype)
        want["dx"] = dx + accumulate
    for n, v in got.items():
        t = dtype if n == "dx" else grads
        _close(v, want[n], bounds[n] + _half_step(np.abs(want[n]) + bounds[n], t), n)
        if v.size >= 1000 and accumulate is None:
            # independent roundings of the projections' gradients and of the result: at most 1 / sqrt(3) of half a step each, in the mean
            rel = np.linalg.norm(v - want[n]) / np.linalg.norm(want[n])
            assert rel <= EPS[dtype] / 2 or dtype == F32, (n, rel)


# M, F, K: one of everything, fewer than a chunk, odd everywhere, a token and a few, one tile and one over, K of one step, of one and a
# bit and of many, tall and wide
SHAPES = [(1, 1, 1), (1, 8, 8), (2, 3, 5), (1, 40, 384), (3, 1024, 384), (7, 129, 65), (16, 64, 64), (17, 65, 72), (33, 200, 1000), (64, 32, 2056),
          (100, 333, 77), (128, 64, 128), (129, 72, 136), (255, 128, 192), (257, 136, 200), (300, 1001, 520), (1000, 96, 40), (2100, 130, 64), (520, 2048, 264)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("M,F,K", SHAPES)
def test_forward(device, M, F, K, dtype):
    for i, gate in enumerate(GATES):
        p = _inputs(400 + i, M, F, K, dtype, bias=i % 2 == 0)
        got = _forward(device, p, dtype, gate)
        _check_forward(p, got, dtype, gate)
        alone, _ = _forward(device, p, dtype, gate, keep=False)
        assert np.array_equal(alone, got[0])
        _check_forward(p, _forward(device, p, dtype, gate, offset=1), dtype, gate)


# the kernels that a forward pass chooses between, each at shapes that it may not be chosen for
WAYS = [("16", "1"), ("64", "1"), ("64", "3"), ("128", "1"), ("256", "1")]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("M,F,K", [(1, 1, 1), (5, 3, 7), (1, 100, 130), (16, 16, 32), (17, 40, 1000), (65, 33, 264), (130, 129, 65), (260, 140, 520), (300, 70, 777)])
def test_forward_every_way(device, monkeypatch, M, F, K, dtype):
    p = _inputs(430, M, F, K, dtype)
    for tile, splits in WAYS:
        monkeypatch.setenv("MOGRAD_HIP_GATED_TILE", tile)
        monkeypatch.setenv("MOGRAD_HIP_GATED_SPLITS", splits)
        for gate in ("silu", "gelu", "relu"):
            for offset in (0, 1):
                _check_forward(p, _forward(device, p, dtype, gate, offset=offset), dtype, gate)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,grads", [(F32, F32), (F16, F16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("M,F,K", SHAPES)
def test_backward(device, M, F, K, dtype, grads):
    for i, gate in enumerate(GATES):
        p = _inputs(410 + i, M, F, K, dtype)
        _check_backward(p, _backward(device, p, dtype, grads, gate, offset=i % 2), dtype, grads, gate)
    old = round_to_dtype(normal(420, 0, (M, K)), dtype)
    _check_backward(p, _backward(device, p, dtype, grads, gate, accumulate=old), dtype, grads, gate, old)
    _check_backward(p, _backward(device, p, dtype, grads, gate, dx=False, db=False), dtype, grads, gate)


@pytest.mark.gpu
@pytest.mark.parametrize("M,F,K", [(1, 1, 1), (5, 3, 7), (70, 100, 130), (129, 65, 33), (260, 140, 264), (1030, 70, 129), (300, 301, 77)])
def test_backward_every_way(device, monkeypatch, M, F, K):
    """fp32: any Linear backward's kernels, and products of bf16 numbers in either tile and with ranges of rows."""
    p = _inputs(431, M, F, K, F32)
    pending = C.c_void_p()
    device.lib.mg_deferred_create(C.byref(pending))
    for tile, splits in (("64", "1"), ("128", "1"), ("128", "3"), ("256", "1"), ("256", "5")):
        monkeypatch.setenv("MOGRAD_HIP_GATED_BWD_TILE", tile)
        monkeypatch.setenv("MOGRAD_HIP_GATED_SPLITS", splits)
        for gate in ("silu", "gelu_tanh"):
            for offset in (0, 1):
                _check_backward(p, _backward(device, p, F32, F32, gate, offset=offset), F32, F32, gate)
        old = round_to_dtype(normal(432, 0, (M, K)), F32)
        _check_backward(p, _backward(device, p, F32, F32, gate, accumulate=old), F32, F32, gate, old)
        got = _backward(device, p, F32, F32, gate, dx=False, db=False)
        _check_backward(p, got, F32, F32, gate)
        later = _backward(device, p, F32, F32, gate, pending=pending)
        assert np.array_equal(later["dw"], _backward(device, p, F32, F32, gate)["dw"])
        _check_backward(p, later, F32, F32, gate)
    device.lib.mg_deferred_destroy(pending)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-25, 1e15])
def test_fp32_far_from_one(device, monkeypatch, size):
    """Products of bf16 numbers keep fp32's digits and range."""
    p = _inputs(433, 150, 70, 100, F32, bias=False)
    p["x"] = (p["x"] * np.float32(size)).astype(np.float32)
    p["w"] = (p["w"] / np.float32(size)).astype(np.float32)
    for tile in ("128", "256"):
        monkeypatch.setenv("MOGRAD_HIP_GATED_TILE", tile)
        _check_forward(p, _forward(device, p, F32, "silu"), F32, "silu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("M,F,K", [(5, 24, 40), (700, 200, 384), (2000, 100, 77), (3000, 500, 300)])
def test_deferred_sums_are_the_immediate_ones(device, M, F, K, dtype):
    p = _inputs(421, M, F, K, dtype)
    pending = C.c_void_p()
    device.lib.mg_deferred_create(C.byref(pending))
    for grads in {dtype, F32}:
        want = _backward(device, p, dtype, grads, "silu")
        got = _backward(device, p, dtype, grads, "silu", pending=pending)
        for n in want:
            assert np.array_equal(got[n], want[n]), n
    device.lib.mg_deferred_destroy(pending)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("gate", GATES)
def test_far_values(device, gate, dtype):
    """Gates far out on either side neither overflow on the way nor become NaN."""
    M, F, K = 24, 16, 8
    p = _inputs(422, M, F, K, dtype)
    far = np.array([-60000.0, -1000.0, -100.0, -30.0, -9.0, -5.0, -0.0, 0.0, 1e-7, 5.0, 9.0, 30.0, 100.0, 1000.0, 6.0, 60000.0], np.float32)
    p["gu"][:, :F] = far
    p["gu"] = round_to_dtype(p["gu"] * 1.0, dtype)
    p["dy"] = round_to_dtype(p["dy"] * 0.01, dtype)
    _check_backward(p, _backward(device, p, dtype, dtype, gate), dtype, dtype, gate)
    p["x"][:] = 0
    p["x"][:, 0] = 1
    p["w"][:, 1:] = 0
    p["w"][:F, 0] = p["gu"][0, :F]
    p["bias"][:F] = 0
    p["w"][F:], p["bias"][F:] = round_to_dtype(0.2 * p["w"][F:], dtype), 0  # (y within fp16)
    _check_forward(p, _forward(device, p, dtype, gate), dtype, gate)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
def test_rows_do_not_touch_each_other(device, dtype):
    """A row of NaNs is that row's, also where tiles read on past the last one."""
    p = _inputs(423, 70, 72, 40, dtype)
    want, _ = _forward(device, p, dtype, "silu")
    p["x"][[3, 69]] = np.nan
    got, _ = _forward(device, p, dtype, "silu")
    rest = np.setdiff1d(np.arange(70), [3, 69])
    assert np.array_equal(got[rest], want[rest]) and np.isnan(got[[3, 69]]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("grads", [BF16, F32])
def test_no_rows(device, grads):
    dw, db = AnyBuffer.create(grads, device, 2 * 8 * 4, fill=3.0), AnyBuffer.create(grads, device, 16, fill=3.0)
    device.lib.mg_gated_linear_bwd(None, None, None, None, None, _ptr(dw), _ptr(db), 0, 8, 4, 0, 0, BF16, grads, device.stream)
    assert (dw.to_numpy() == 0).all() and (db.to_numpy() == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("M,F,K", [(600, 136, 200), (77, 101, 33)])
def test_forward_then_backward(device, dtype, M, F, K):
    """The two as they are used together: the backward reads what the forward kept."""
    p = _inputs(424, M, F, K, dtype)
    _, p["gu"] = _forward(device, p, dtype, "silu")
    _check_backward(p, _backward(device, p, dtype, dtype, "silu"), dtype, dtype, "silu")


@pytest.mark.gpu
def test_twice_gives_the_same_bits(device):
    p = _inputs(425, 3000, 256, 384, BF16)
    a, b = (_backward(device, p, BF16, F32, "silu") for _ in range(2))
    for n in a:
        assert np.array_equal(a[n], b[n]), n
    assert np.array_equal(_forward(device, p, BF16, "silu")[0], _forward(device, p, BF16, "silu")[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M,F,K", [(1, 1, 8), (3, 40, 24), (37, 130, 16), (300, 1001, 64), (2100, 136, 40), (5000, 1024, 8), (4097, 77, 9)])
def test_bias_gradients_are_sums_of_unrounded_values(device, M, F, K, dtype):
    """db is rounded once, as its own type: none of the rounding of the projections' gradients is in it."""
    for i, gate in enumerate(GATES):
        p = _inputs(640 + i, M, F, K, dtype, bias=False)
        _, _, db, d = O.gated_linear_bwd(p["dy"], p["gu"], p["x"], p["w"], gate)
        act_off, slope_off = _act_error(p["gu"][:, :F].astype(np.float64), gate, 0.0)
        dy = np.abs(p["dy"])
        off = np.concatenate([dy * np.abs(p["gu"][:, F:]) * slope_off, dy * act_off], axis=1) + 4 * U * np.abs(d)
        bound = off.sum(0) + (M + 16) * U * (np.abs(d) + off).sum(0)
        for grads in (dtype, F32):
            got = _backward(device, p, dtype, grads, gate)["db"]
            _close(got, db, bound + _half_step(np.abs(db) + bound, grads), "db")
