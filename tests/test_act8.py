"""Activations in 8 bits: the format, a Linear layer's gradients from it.

The format's numbers are exact (a step is a power of two), so what is stored and what comes back is compared for equality.
The Linear gradients are products of the restored values: compared with float64 products of the same numbers.
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


# ---- the format itself (the oracle), no GPU ------------------------------------------------


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_the_step_is_the_least_that_fits(kind):
    """Against a search over every step."""
    lo, hi = O.ACT8_RANGE[kind]
    rng = np.random.default_rng(3)
    x = np.ldexp(rng.standard_normal((64, 70)), rng.integers(lo + 12, hi + 3, (64, 1)))
    x[0] = 0
    x[1, :32] = np.ldexp(127.5, 3 if kind != "f16" else 2)   # rounds to 128 at the step it would have: the next one
    x[2, :32] = np.ldexp(127.4999, 3 if kind != "f16" else 2)
    act8 = O.act8_store(x, kind)
    rows, cols = x.shape
    blocks = 3
    q = act8[:rows * blocks * 32].view(np.int8).reshape(rows, blocks, 32)
    k = act8[rows * blocks * 32:].reshape(rows, blocks).astype(int) - 133
    padded = np.zeros((rows, blocks * 32))
    padded[:, :cols] = x
    padded = padded.reshape(rows, blocks, 32)
    for r in range(rows):
        for b in range(blocks):
            fits = [s for s in range(lo, hi + 1) if np.abs(np.rint(np.ldexp(padded[r, b], -s))).max() <= 127]
            step = fits[0] if fits else hi
            assert k[r, b] == step
            assert np.array_equal(q[r, b], np.clip(np.rint(np.ldexp(padded[r, b], -step)), -127, 127))
    assert np.abs(O.act8_load(act8, rows, cols) - x).max() <= np.ldexp(0.5, k.max()) or hi == k.max()


def test_whole_numbers_are_their_own_8_bits():
    x = np.arange(-127, 128, dtype=np.float64).reshape(1, -1)
    x = np.concatenate([x, np.full((1, 1), 127.0)], axis=1).reshape(-1, 32)
    assert np.array_equal(O.act8_load(O.act8_store(x, "bf16"), *x.shape), x)


def test_bytes():
    lib = mograd_amd.load()
    for rows, cols in [(1, 1), (1, 32), (3, 33), (16384, 1536), (7, 1001)]:
        assert lib.mg_act8_bytes(rows, cols) == len(O.act8_store(np.zeros((rows, cols)), "f32"))
    assert lib.mg_act8_bytes(0, 5) == 0 and lib.mg_act8_bytes(5, 0) == 0 and lib.mg_act8_bytes(-1, 5) == 0
    assert lib.mg_act8_bytes(1 << 31, 32) == 0
    assert lib.mg_act8_bytes(1 << 20, 1 << 20) == (1 << 40) + (1 << 35)


def test_refusals():
    """Answered before anything is launched; the pointers are never followed."""
    lib = mograd_amd.load()
    p = C.c_void_p(4096)
    odd = C.c_void_p(4100)
    store = lambda x, a, rows, cols, dtype: lib.mg_act8_store(x, a, rows, cols, 0, dtype, None)
    load = lambda x, a, rows, cols, dtype: lib.mg_act8_load(a, x, rows, cols, dtype, None)
    for call in (store, load):
        for args in [(p, p, 4, 4, I32), (p, p, 4, 4, 9), (p, p, -1, 4, F32), (p, p, 4, 0, F32), (None, p, 4, 4, F32),
                     (p, None, 4, 4, F32), (p, odd, 4, 4, F32), (p, p, 1 << 31, 4, F32), (p, p, 1 << 30, 1 << 29, F32)]:
            with pytest.raises(MogradError) as e:
                call(*args)
            assert e.value.status == 1 and "act8" in str(e.value)
        assert call(p, p, 0, 4, F32) == 0  # nothing to do

    def linear(dy=p, x8=p, w=p, dx=p, dw=p, M=4, N=4, K=4, dtype=BF16, grads=BF16):
        return lib.mg_linear_bwd_act8(dy, x8, w, dx, dw, None, M, N, K, 0, 0, dtype, grads, None)

    for bad in [dict(dtype=I64), dict(grads=F16), dict(dtype=F32, grads=BF16), dict(M=-1), dict(N=0), dict(K=0), dict(dy=None),
                dict(x8=None), dict(w=None), dict(dw=None), dict(x8=odd)]:
        with pytest.raises(MogradError) as e:
            linear(**bad)
        assert e.value.status == 1 and "linear_bwd_act8" in str(e.value)


# ---- storing and restoring on the GPU ------------------------------------------------------


def _bytes(device, n, fill=0xA5):
    """A device buffer of n bytes (rounded up to 4) with a known filling."""
    words = -(-n // 4) + 4
    return AnyBuffer.from_numpy(device, np.full(words, int.from_bytes(bytes([fill] * 4), "little", signed=True), np.int32), I32)


def _upload(device, data):
    data = np.ascontiguousarray(data, np.uint8)
    padded = np.zeros(-(-len(data) // 4) * 4, np.uint8)
    padded[:len(data)] = data
    return AnyBuffer.from_numpy(device, padded.view(np.int32), I32)


def _download(buf):
    return buf.to_numpy().view(np.uint8)


def _values(seed, rows, cols, dtype):
    x = normal(seed, 0, (rows, cols)) * np.exp(normal(seed, 1, (1, cols)))
    x = round_to_dtype(x, dtype)
    x[0, :] = 0
    if rows > 2:
        x[1] = np.abs(x[1])
        x[2] *= np.float32(2.0 ** -9)
    return round_to_dtype(x, dtype)


SHAPES = [(1, 1), (2, 7), (5, 31), (5, 32), (5, 33), (3, 64), (33, 100), (17, 384), (9, 1001), (4, 4104), (1, 70000), (5000, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("keep_sign", [0, 1])
def test_store_and_load(device, dtype, rows, cols, keep_sign):
    x = _values(11, rows, cols, dtype)
    want = O.act8_store(x, KIND[dtype], bool(keep_sign))
    lib, n = device.lib, len(want)
    for offset in (0, 1):  # and a tensor that starts off the 16-byte chunks
        src = AnyBuffer.from_numpy(device, np.concatenate([np.zeros(offset, np.float32), x.reshape(-1)]), dtype)
        act8 = _bytes(device, n)
        lib.mg_act8_store(AnyBuffer(src.storage, dtype, rows * cols, offset).data_ptr(), act8.data_ptr(), rows, cols, keep_sign,
                          dtype, device.stream)
        got = _download(act8)
        assert np.array_equal(got[:n], want)
        assert (got[n:] == 0xA5).all()
        back = AnyBuffer.create(dtype, device, offset + rows * cols + 3, fill=7.0)
        lib.mg_act8_load(act8.data_ptr(), AnyBuffer(back.storage, dtype, rows * cols, offset).data_ptr(), rows, cols, dtype,
                         device.stream)
        b = back.to_numpy()
        assert np.array_equal(b[offset:offset + rows * cols].reshape(rows, cols), O.act8_load(want, rows, cols))
        assert (b[:offset] == 7).all() and (b[offset + rows * cols:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
def test_extremes(device, dtype):
    """The type's largest and least values, halfway cases, zeros of both signs, infinities and NaN."""
    big = {F32: np.float32(3.4028235e38), BF16: np.float32(3.3895314e38), F16: np.float32(65504)}[dtype]
    tiny = {F32: np.float32(1e-45), BF16: np.float32(9.2e-41), F16: np.float32(6e-8)}[dtype]
    x = np.zeros((12, 64), np.float32)
    x[0, 0], x[0, 1] = big, -big
    x[1, :3] = tiny, -tiny, 0
    x[2, :8] = 127, 63.5, 62.5, 0.5, 1.5, -0.5, -62.5, 0.25
    x[3, :4] = 127.5, 64.0, 1.0, -1.0
    x[4, 5] = np.inf
    x[5, 40] = -np.inf
    x[6, 3] = np.nan
    x[7] = -0.0
    x[8, :2] = 65280, 65216
    x[9, 0], x[9, 1] = 1, tiny
    x[10, 0], x[10, 63] = 2.0 ** -13, 2.0 ** 13
    x = round_to_dtype(x, dtype)
    lib = device.lib
    for keep_sign in (0, 1):
        want = O.act8_store(x, KIND[dtype], bool(keep_sign))
        src = AnyBuffer.from_numpy(device, x, dtype)
        act8 = _bytes(device, len(want))
        lib.mg_act8_store(src.data_ptr(), act8.data_ptr(), *x.shape, keep_sign, dtype, device.stream)
        assert np.array_equal(_download(act8)[:len(want)], want)
        back = AnyBuffer.create(dtype, device, x.size)
        lib.mg_act8_load(act8.data_ptr(), back.data_ptr(), *x.shape, dtype, device.stream)
        values = O.act8_load(want, *x.shape)
        np.testing.assert_array_equal(back.to_numpy(x.shape), values)
        assert np.isnan(values[4, :32]).all() and not np.isnan(values[4, 32:]).any()
        if keep_sign:
            assert np.array_equal((values > 0)[:4], (x > 0)[:4]) and values[9, 1] > 0


# ---- a Linear layer's gradients ------------------------------------------------------------


def _linear(device, dy, act8, w, M, N, K, dtype, grads, relu=0, accumulate=None, with_dx=True, with_db=True, offset=0):
    place = lambda a, t: AnyBuffer.from_numpy(device, np.concatenate([np.zeros(offset, np.float32), np.asarray(a, np.float32).reshape(-1)]), t)
    shifted = lambda b, n: AnyBuffer(b.storage, b.dtype, n, offset).data_ptr()
    bdy, bw, b8 = place(dy, dtype), place(w, dtype), _upload(device, act8)
    dx = place(accumulate if accumulate is not None else np.full((M, K), 3.0), dtype) if with_dx else None
    dw = place(np.full((N, K), 5.0), grads)
    db = place(np.full(N, 5.0), grads) if with_db else None
    device.lib.mg_linear_bwd_act8(shifted(bdy, M * N), b8.data_ptr(), shifted(bw, N * K) if with_dx else None,
                                  shifted(dx, M * K) if with_dx else None, shifted(dw, N * K), shifted(db, N) if with_db else None,
                                  M, N, K, int(accumulate is not None), relu, dtype, grads, device.stream)
    cut = lambda b, shape: b.to_numpy()[offset:].reshape(shape)
    return cut(dx, (M, K)) if with_dx else None, cut(dw, (N, K)), cut(db, (N,)) if with_db else None


def _bound(want, mass, terms, dtype, extra=0.0):
    """Half a step of the output type, and fp32 sums of `terms` products of total magnitude `mass`: partial sums in any order
    lose at most one rounding, 2^-24, of the mass for each addition that a value goes through.  The matrix cores and the
    partial sums give chains of no more than `terms`; rounding errors of random sign grow with its root, and eight times
    that is allowed.  (Half a step of fp16 is never less than 2^-25, half of its spacing below 2^-14.)"""
    chain = 16 + 8 * np.sqrt(terms)
    return np.maximum(EPS[dtype] / 2 * np.abs(want), 2.0 ** -25 if dtype == F16 else 0.0) + 2.0 ** -24 * chain * mass + extra


def _check(got, want, bound, what):
    assert np.isfinite(got).all(), what
    worst = float((np.abs(got - want) / np.maximum(bound, 1e-300)).max())
    assert worst <= 1, f"{what}: {worst:.3g} of the bound"


LINEARS = [(1, 1, 1), (1, 5, 3), (7, 33, 20), (64, 64, 64), (100, 96, 130), (257, 65, 384), (128, 1001, 77), (999, 40, 32),
           (513, 256, 300), (3000, 130, 136), (1024, 384, 768), (2048, 512, 2048), (4097, 384, 384), (1999, 1001, 768)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,grads", [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32), (F32, F32)])
@pytest.mark.parametrize("M,N,K", LINEARS)
@pytest.mark.parametrize("relu", [0, 1])
@pytest.mark.parametrize("route,splits", [("", ""), ("1", "1"), ("1", "5")])
def test_linear_gradients(device, monkeypatch, M, N, K, dtype, grads, relu, route, splits):
    """By the choice that is made for the size, and by the tiles that multiply the bytes, in one range of rows and in several."""
    monkeypatch.setenv("MOGRAD_HIP_ACT8_ROUTE", route)
    monkeypatch.setenv("MOGRAD_HIP_ACT8_SPLITS", splits)
    x = _values(21, M, K, dtype)
    if relu:
        x = np.maximum(x, 0)
    act8 = O.act8_store(x, KIND[dtype], bool(relu))
    x8 = O.act8_load(act8, M, K)
    if relu:
        assert np.array_equal(x8 > 0, x > 0)
    dy = round_to_dtype(normal(21, 3, (M, N), std=0.1), dtype).astype(np.float64)
    w = round_to_dtype(normal(21, 4, (N, K), std=K ** -0.5), dtype).astype(np.float64)
    before = round_to_dtype(normal(21, 5, (M, K)), dtype)
    for accumulate, offset in ((None, 0), (before, 1)):
        dx, dw, db = _linear(device, dy, act8, w, M, N, K, dtype, grads, relu, accumulate, offset=offset)
        want = dy @ w * ((x8 > 0) if relu else 1)
        bound = _bound(want, np.abs(dy) @ np.abs(w), N, dtype)
        if accumulate is not None:  # the product is rounded, then the sum
            want = want + before
            bound = bound + EPS[dtype] / 2 * (np.abs(want) + bound)
        _check(dx, want, bound, "dx")
        want = dy.T @ x8
        _check(dw, want, _bound(want, np.abs(dy).T @ np.abs(x8), M, grads), "dw")
        _check(db, dy.sum(0), _bound(dy.sum(0), np.abs(dy).sum(0), M, grads), "db")


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(4097, 36, 132), (1000, 100, 580), (2500, 512, 260)])
@pytest.mark.parametrize("tile", ["0", "64", "128"])
@pytest.mark.parametrize("relu", [0, 1])
@pytest.mark.parametrize("accumulate", [False, True])
def test_f32_dx_beside_dw(device, monkeypatch, M, N, K, tile, relu, accumulate):
    """fp32 arrays on 16-byte chunks: dx in the launch of dw, by either tile, and in one of its own; masked where x is not positive, or
    was not finite."""
    monkeypatch.setenv("MOGRAD_HIP_ACT8_ROUTE", "1")
    monkeypatch.setenv("MOGRAD_HIP_ACT8_XTILE", tile)
    x = _values(26, M, K, F32)
    if relu:
        x = np.maximum(x, 0)
        x[M // 2, 40] = np.inf
    act8 = O.act8_store(x, "f32", bool(relu))
    x8 = O.act8_load(act8, M, K)
    dy = normal(26, 3, (M, N), std=0.1).astype(np.float32).astype(np.float64)
    w = normal(26, 4, (N, K), std=K ** -0.5).astype(np.float32).astype(np.float64)
    before = normal(26, 5, (M, K)).astype(np.float32) if accumulate else None
    dx, dw, db = _linear(device, dy, act8, w, M, N, K, F32, F32, relu, before)
    with np.errstate(invalid="ignore"):
        want = dy @ w * ((x8 > 0) if relu else 1)
    bound = _bound(want, np.abs(dy) @ np.abs(w), N, F32)
    if accumulate:
        want = want + before
        bound = bound + EPS[F32] / 2 * (np.abs(want) + bound)
    _check(dx, want, bound, "dx")
    rest = np.r_[0:32, 64:K] if relu else np.arange(K)
    if relu:
        assert (dx[M // 2, 32:64] == (before[M // 2, 32:64] if accumulate else 0)).all() and np.isnan(dw[:, 32:64]).all()
    want = dy.T @ x8[:, rest]
    _check(dw[:, rest], want, _bound(want, np.abs(dy).T @ np.abs(x8[:, rest]), M, F32), "dw")
    _check(db, dy.sum(0), _bound(dy.sum(0), np.abs(dy).sum(0), M, F32), "db")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_linear_without_dx_or_db(device, dtype):
    M, N, K = 300, 72, 200
    x = _values(22, M, K, dtype)
    act8 = O.act8_store(x, KIND[dtype])
    dy = round_to_dtype(normal(22, 3, (M, N)), dtype)
    w = round_to_dtype(normal(22, 4, (N, K)), dtype)
    full = _linear(device, dy, act8, w, M, N, K, dtype, F32)
    some = _linear(device, dy, act8, w, M, N, K, dtype, F32, with_dx=False, with_db=False)
    want = dy.astype(np.float64).T @ O.act8_load(act8, M, K)
    mass = np.abs(dy).T.astype(np.float64) @ np.abs(x)
    for dw in (full[1], some[1]):
        _check(dw, want, _bound(want, mass, M, F32), "dw")


@pytest.mark.gpu
def test_linear_of_no_rows(device):
    dw = AnyBuffer.create(F32, device, 6, fill=4.0)
    db = AnyBuffer.create(F32, device, 2, fill=4.0)
    device.lib.mg_linear_bwd_act8(None, None, None, None, dw.data_ptr(), db.data_ptr(), 0, 2, 3, 0, 0, BF16, F32, device.stream)
    assert (dw.to_numpy() == 0).all() and (db.to_numpy() == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("route", ["0", "1"])
def test_what_was_not_finite_shows_in_the_gradient(device, monkeypatch, dtype, route):
    """An infinity in the forward's activation: NaN in the columns of dw of its block, the other columns as ever."""
    monkeypatch.setenv("MOGRAD_HIP_ACT8_ROUTE", route)
    M, N, K = 130, 48, 160
    x = _values(23, M, K, dtype)
    clean = O.act8_load(O.act8_store(x, KIND[dtype]), M, K)
    x[77, 70] = np.inf
    act8 = O.act8_store(x, KIND[dtype])
    dy = round_to_dtype(normal(23, 3, (M, N)), dtype).astype(np.float64)
    _, dw, _ = _linear(device, dy, act8, np.zeros((N, K)), M, N, K, dtype, F32)
    assert np.isnan(dw[:, 64:96]).all()
    rest = np.r_[0:64, 96:160]
    want = dy.T @ clean[:, rest]
    _check(dw[:, rest], want, _bound(want, np.abs(dy).T @ np.abs(clean[:, rest]), M, F32), "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("M,N,K", [(64, 8, 32), (190, 131, 129), (130, 256, 96)])
def test_large_and_infinite_gradients(device, monkeypatch, dtype, M, N, K):
    """The largest finite dY, tiny ones and an infinity, by the tiles that multiply the bytes: what fp32 products would give."""
    monkeypatch.setenv("MOGRAD_HIP_ACT8_ROUTE", "1")
    big = {F32: np.float32(3.4028235e38), BF16: np.float32(3.3895314e38), F16: np.float32(65504)}[dtype]
    x = np.zeros((M, K), np.float32)
    x[::7, ::5] = 0.5
    x[5, 1] = 2.0
    act8 = O.act8_store(x, KIND[dtype])
    assert np.array_equal(O.act8_load(act8, M, K), x)
    dy = np.zeros((M, N), np.float32)
    dy[7, 0], dy[14, 1], dy[21, 2], dy[28, 3] = big, -big, np.inf, np.float32(2.0 ** -24)
    dy[5, 4] = np.float32(1 + 2.0 ** -23) if dtype == F32 else 1.0
    dy = round_to_dtype(dy, dtype)
    _, dw, db = _linear(device, dy, act8, np.zeros((N, K)), M, N, K, dtype, F32)
    with np.errstate(invalid="ignore"):
        want = (dy.astype(np.float64)[:, :, None] * x.astype(np.float64)[:, None, :]).sum(axis=0)
    np.testing.assert_array_equal(dw, want.astype(np.float32))
    np.testing.assert_array_equal(db, dy.astype(np.float64).sum(axis=0).astype(np.float32))


@pytest.mark.gpu
def test_routes_agree(device, monkeypatch):
    """The restored copy and the bytes are the same numbers: the results are, up to the order of the sums."""
    for dtype in FLOATS:
        M, N, K = 1500, 264, 200
        act8 = O.act8_store(np.maximum(_values(25, M, K, dtype), 0), KIND[dtype], True)
        dy = round_to_dtype(normal(25, 3, (M, N)), dtype)
        w = round_to_dtype(normal(25, 4, (N, K)), dtype)
        runs = []
        for route in ("0", "1"):
            monkeypatch.setenv("MOGRAD_HIP_ACT8_ROUTE", route)
            runs.append(_linear(device, dy, act8, w, M, N, K, dtype, F32, relu=1))
        x8, a = O.act8_load(act8, M, K), np.abs(dy.astype(np.float64))
        assert (runs[0][0] == 0).sum() == (runs[1][0] == 0).sum() >= (x8 <= 0).sum()
        for i, mass in ((0, a @ np.abs(w.astype(np.float64))), (1, a.T @ np.abs(x8)), (2, a.sum(0))):
            bound = _bound(runs[0][i], mass, max(M, N), dtype if i == 0 else F32)
            assert (np.abs(runs[0][i].astype(np.float64) - runs[1][i]) <= 2 * bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("route", ["0", "1"])
def test_linear_twice_gives_the_same_bits(device, monkeypatch, dtype, route):
    monkeypatch.setenv("MOGRAD_HIP_ACT8_ROUTE", route)
    M, N, K = 2000, 96, 160
    act8 = O.act8_store(_values(24, M, K, dtype), KIND[dtype])
    dy = round_to_dtype(normal(24, 3, (M, N)), dtype)
    w = round_to_dtype(normal(24, 4, (N, K)), dtype)
    a = _linear(device, dy, act8, w, M, N, K, dtype, F32)
    b = _linear(device, dy, act8, w, M, N, K, dtype, F32)
    for u, v in zip(a, b):
        assert np.array_equal(u, v)
