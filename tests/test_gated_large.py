"""Gated layers, rotary positions and clipping where elements are counted past 2^31: what lies in the first, the last and other rows."""
import ctypes as C

import numpy as np
import pytest

from helpers import normal
from oracle import oracle_np as O
from test_gated_linear import _check_forward
from test_residual_norm import U, _close, _half_step

pytestmark = pytest.mark.gpu

from mograd_amd import BF16, F32, AnyBuffer  # noqa: E402
from mograd_amd.runtime import round_to_dtype  # noqa: E402


def _rows(buf, rows, cols):
    """Some rows of a large (.., cols) buffer."""
    return np.stack([AnyBuffer(buf.storage, buf.dtype, cols, int(r) * cols).to_numpy() for r in rows])


@pytest.mark.parametrize("dtype,tile", [(BF16, "64"), (BF16, "128"), (BF16, "256"), (BF16, None), (F32, "128"), (F32, None)])
def test_gated_layer(device, monkeypatch, dtype, tile):
    M, F, K = 140000, 8192, 16  # 2.3e9 projections
    if tile:
        monkeypatch.setenv("MOGRAD_HIP_GATED_TILE", tile)
    p = {"x": round_to_dtype(normal(800, 0, (M, K)), dtype), "w": round_to_dtype(normal(800, 1, (2 * F, K), 0.3), dtype), "bias": None}
    x, w = (AnyBuffer.from_numpy(device, p[n], dtype) for n in ("x", "w"))
    y, gu = AnyBuffer.create(dtype, device, M * F), AnyBuffer.create(dtype, device, M * 2 * F)
    device.lib.mg_gated_linear_fwd(x.data_ptr(), w.data_ptr(), None, y.data_ptr(), gu.data_ptr(), M, F, K, 0, dtype, device.stream)
    rows = np.array([0, 1, 65535, 65536, 131071, 131072, 131073, M - 2, M - 1])
    _check_forward({**p, "x": p["x"][rows]}, (_rows(y, rows, F), _rows(gu, rows, 2 * F)), dtype, "silu")
    if tile:
        return
    # the gradients of dy = 0.25: dx of some rows, dw of some columns
    del y
    dy = AnyBuffer.create(dtype, device, M * F, fill=0.25)
    dx, dw, db = AnyBuffer.create(dtype, device, M * K), AnyBuffer.create(F32, device, 2 * F * K), AnyBuffer.create(F32, device, 2 * F)
    device.lib.mg_gated_linear_bwd(dy.data_ptr(), gu.data_ptr(), x.data_ptr(), w.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(), M, F, K, 0, 0, dtype,
                                   F32, device.stream)
    kept = _rows(gu, rows, 2 * F)
    want, _, _, d = O.gated_linear_bwd(np.full((len(rows), F), 0.25), kept, p["x"][rows], p["w"], "silu")
    mass = np.abs(d) @ np.abs(p["w"]).astype(np.float64)
    half = {BF16: 2.0 ** -8, F32: 64 * U}[dtype]  # of each term: its rounding, or the act's few units
    _close(_rows(dx, rows, K), want, _half_step(want, dtype) + (half + 2 * F * U) * mass, "dx")
    cols = np.array([0, 1, 4097, F - 1])
    got = dw.to_numpy().reshape(2 * F, K)[np.concatenate([cols, F + cols])]
    pair = np.concatenate([cols, F + cols])
    # (what the backward read: the projections as they were stored, a rounding away from these)
    _, kept = O.gated_linear_fwd(p["x"], p["w"][pair], None, "silu")
    want, dwant, dbwant, d = O.gated_linear_bwd(np.full((M, len(cols)), 0.25), round_to_dtype(kept, dtype), p["x"], p["w"][pair], "silu")
    terms = np.abs(d).T @ np.abs(p["x"]).astype(np.float64)
    # a projection that fp32 rounds the other way is one step off, and its gradient with it
    bound = (4 * half + M * U) * terms
    _close(got, dwant, bound, "dw")
    _close(db.to_numpy()[pair], dbwant, (4 * half + M * U) * np.abs(d).sum(0), "db")


def test_rotary(device):
    S, H, D = 70000, 512, 64  # 2.3e9 values, all 1
    x = AnyBuffer.create(BF16, device, S * H * D, fill=1.0)
    freq = (1e4 ** (-np.arange(D // 2) / (D // 2))).astype(np.float32)
    f, st = AnyBuffer.from_numpy(device, freq, F32), (C.c_int64 * 3)(S * H * D, H * D, D)
    device.lib.mg_rotary(x.data_ptr(), x.data_ptr(), None, f.data_ptr(), None, 1, S, H, D, D, st, st, None, 1, 0, 0, 0, BF16, device.stream)
    rows = np.array([0, 1, 65535, 65536, 65537, S - 1])
    got = _rows(x, rows, H * D).reshape(len(rows), H, D)
    want, _ = O.rotary(np.ones((1, len(rows), 1, D)), rows.reshape(1, 1, -1), freq, [0] * (D // 2))
    want = np.broadcast_to(want[0], got.shape)
    _close(got, want, _half_step(want, BF16) + 12 * U, "y")


@pytest.mark.parametrize("in_place", [False, True])
def test_clipping(device, in_place):
    n = 2 ** 31 + 4099
    g = AnyBuffer.create(BF16, device, n, fill=0.5)
    out = g if in_place else AnyBuffer.create(BF16, device, n, fill=3.0)
    norm = AnyBuffer.create(F32, device, 1)
    most = 0.25 * np.sqrt(n)
    arrays = (C.c_void_p * 1)(g.data_ptr().value), (C.c_void_p * 1)(out.data_ptr().value), (C.c_int64 * 1)(n), (C.c_int * 1)(BF16)
    device.lib.mg_clip_grads(*arrays, 1, most, norm.data_ptr(), device.stream)
    want = 0.5 * np.sqrt(n)
    assert abs(norm.to_numpy()[0] - want) <= 2 * U * want
    for at in (0, 2 ** 30, 2 ** 31 - 8, n - 4099, n - 1):
        part = AnyBuffer(out.storage, BF16, min(4099, n - at), at).to_numpy()
        assert (part == 0.25).all(), at
