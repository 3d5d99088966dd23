"""Rotary positions against float64.

Tolerance, per value: half a step of the output's type, and of the pair's magnitude |a| + |b| six roundings in fp32 (sine and cosine one
and a half each, their products and the sum) and what the angle is off by in 64 bits, 2^-51 of it (two roundings, and two of the oracle's).
"""
import ctypes as C

import numpy as np
import pytest

from helpers import normal
from oracle import oracle_np as O
from test_residual_norm import FLOATS, U, _close, _half_step

import mograd_amd
from mograd_amd import BF16, F16, F32, I32, I64, AnyBuffer, MogradError
from mograd_amd.runtime import round_to_dtype

i64s = lambda *v: (C.c_int64 * len(v))(*v)
i32s = lambda v: (C.c_int32 * len(v))(*v)


def test_oracle():
    """A turn keeps lengths, turns add up, and the inverse is the gradient."""
    rng = np.random.default_rng(1)
    x, dy = rng.standard_normal((2, 5, 3, 12)), rng.standard_normal((2, 5, 3, 12))
    f, axis = rng.random(5), [0, 1, 0, 1, 1]
    p, q = rng.integers(-9, 99, (2, 2, 5)), rng.integers(-9, 99, (2, 2, 5))
    for nb in (False, True):
        y, _ = O.rotary(x, p, f, axis, nb)
        np.testing.assert_allclose(O.rotary(y, q, f, axis, nb)[0], O.rotary(x, p + q, f, axis, nb)[0], atol=1e-12)
        np.testing.assert_allclose(O.rotary(y, p, f, axis, nb, inverse=True)[0], x, atol=1e-12)
        np.testing.assert_allclose((y * dy).sum(), (x * O.rotary(dy, p, f, axis, nb, inverse=True)[0]).sum(), atol=1e-12)
        assert np.array_equal(y[..., 10:], x[..., 10:])
    one = O.rotary(np.ones((1, 2, 1, 2)), [[[0, 1]]], [np.pi / 2], [0])[0]
    np.testing.assert_allclose(one.reshape(2, 2), [[1, 1], [-1, 1]], atol=1e-12)


def test_refusals():
    """Answered before anything is launched; the pointers are never followed."""
    lib = mograd_amd.load()
    p = C.c_void_p(4096)

    def call(x=p, y=p, positions=p, inv_freq=p, axis=i32s([0, 1, 2, 0]), B=2, S=3, H=2, D=16, rotated=8, xs=i64s(96, 32, 16), ys=i64s(96, 32, 16),
             ps=i64s(6, 3, 1), axes=3, pos=I32, dtype=BF16):
        return lib.mg_rotary(x, y, positions, inv_freq, axis, B, S, H, D, rotated, xs, ys, ps, axes, pos, 0, 0, dtype, None)

    for bad in (dict(dtype=I32), dict(dtype=7), dict(B=-1), dict(S=-1), dict(H=-1), dict(D=0), dict(D=6), dict(rotated=0), dict(rotated=7), dict(rotated=-2),
                dict(D=600, rotated=514), dict(B=1 << 41), dict(B=1 << 30, S=1 << 20), dict(xs=None), dict(ys=None), dict(ps=None),
                dict(xs=i64s(-1, 32, 16)), dict(ys=i64s(96, -32, 16)), dict(ys=i64s(96, 32, 0)), dict(ps=i64s(6, 3, -1)), dict(pos=F32), dict(pos=BF16), dict(axes=0),
                dict(axes=256), dict(axes=2), dict(axis=None), dict(axis=i32s([0, -1, 0, 0])), dict(x=None), dict(y=None), dict(inv_freq=None), dict(xs=i64s(192, 64, 16))):
        with pytest.raises(MogradError) as e:
            call(**bad)
        assert e.value.status == 1 and "rotary" in str(e.value), bad
    with pytest.raises(MogradError) as e:
        call(H=1 << 20)
    assert e.value.status == 2
    for empty in (dict(B=0), dict(S=0), dict(H=0)):
        assert call(x=None, y=None, inv_freq=None, **empty) == 0


# ---- on the GPU ----------------------------------------------------------------------------


def _freq(pairs, base=10000.0):
    return (base ** (-np.arange(pairs) / pairs)).astype(np.float32)


class _View:
    """A (B, S, H, D) view into a buffer with gaps of `gap` elements between heads, `offset` elements into it; the gaps are guards."""

    def __init__(self, device, a, dtype, order="bshd", gap=0, offset=0):
        B, S, H, D = a.shape
        row = D + gap
        s, h, b = {"bshd": (H * row, row, S * H * row), "bhsd": (row, S * row, H * S * row)}[order]
        self.shape, self.strides, self.offset, self.dtype, self.device = a.shape, (b, s, h), offset, dtype, device
        host = np.full(offset + B * S * H * row + 9, -3.0, np.float32)
        self.index = (offset + np.arange(B)[:, None, None, None] * b + np.arange(S)[:, None, None] * s + np.arange(H)[:, None] * h + np.arange(D))
        host[self.index] = a
        self.buf = AnyBuffer.from_numpy(device, host, dtype)
        self.ptr = AnyBuffer(self.buf.storage, dtype, B * S * H * row, offset).data_ptr()

    def read(self):
        host = self.buf.to_numpy()
        got = host[self.index]
        host[self.index] = -3
        assert (host == -3).all(), "written between or outside the heads"
        return got


def _run(device, x, y, positions, inv_freq, pair_axis, neighbours, inverse, rotated, pos_dtype=I32, pos_strides=None):
    B, S, H, D = x.shape
    pos = None if positions is None else AnyBuffer.from_numpy(device, positions.astype(np.int32 if pos_dtype == I32 else np.int64))
    freq = AnyBuffer.from_numpy(device, inv_freq, F32)
    axes = 1 if positions is None else len(positions)
    ps = None if positions is None else i64s(*(pos_strides or (B * S, S, 1)))
    device.lib.mg_rotary(x.ptr, y.ptr, None if pos is None else pos.data_ptr(), freq.data_ptr(), None if pair_axis is None else i32s(pair_axis), B, S, H, D,
                         rotated, i64s(*x.strides), i64s(*y.strides), ps, axes, pos_dtype, int(neighbours), int(inverse), x.dtype, device.stream)
    device.synchronize()


def _check(a, got, positions, inv_freq, pair_axis, neighbours, inverse, dtype):
    want, angle = O.rotary(a, positions, inv_freq, pair_axis, neighbours, inverse)
    bound = _half_step(want, dtype)
    c0, c1 = O.rotary_pairs(2 * len(inv_freq), neighbours)
    size = (np.abs(a[..., c0]) + np.abs(a[..., c1])) * (6 * U + 2.0 ** -51 * np.abs(angle))[:, :, None, :]
    bound[..., c0] += size
    bound[..., c1] += size
    _close(got, want, bound, "y")
    rest = slice(2 * len(inv_freq), None)
    assert np.array_equal(got[..., rest], a[..., rest])


# B, S, H, D, rotated: one pair, one token, odd heads and lengths, widths of no whole chunk, rests of every kind, the most pairs, more
# tokens than one workgroup's
SHAPES = [(1, 1, 1, 2, 2), (2, 1, 3, 8, 8), (1, 7, 1, 50, 50), (3, 5, 2, 66, 64), (2, 33, 6, 64, 64), (1, 130, 5, 80, 40), (2, 65, 4, 128, 64), (1, 9, 3, 512, 512),
          (1, 4, 2, 600, 512), (2, 3, 1, 96, 2), (5, 77, 2, 32, 32), (1, 1025, 2, 96, 96), (2, 600, 1, 20, 12), (1, 3, 40, 256, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("B,S,H,D,rotated", SHAPES)
def test_against_float64(device, B, S, H, D, rotated, dtype):
    a = round_to_dtype(normal(500, 0, (B, S, H, D), 2.0), dtype)
    pairs = rotated // 2
    rng = np.random.default_rng(pairs)
    for i, (axes, neighbours, inverse, order, gap, offset, pos_dtype) in enumerate((
            (1, 0, 0, "bshd", 0, 0, I32), (3, 1, 1, "bshd", 8, 8, I64), (2, 0, 1, "bhsd", 3, 1, I32), (3, 1, 0, "bhsd", 0, 0, I64), (5, 0, 0, "bshd", 16, 1, I64))):
        positions = rng.integers(-3, 70, (axes, B, S)) + np.arange(S) + (1 << 20) * (i % 2)
        pair_axis = list(rng.integers(0, axes, pairs)) if axes > 1 else None
        x, y = _View(device, a, dtype, order, gap, offset), _View(device, np.full_like(a, 7.0), dtype)
        _run(device, x, y, positions, _freq(pairs), pair_axis, neighbours, inverse, rotated, pos_dtype)
        _check(a, y.read(), positions, _freq(pairs), pair_axis or [0] * pairs, neighbours, inverse, dtype)
        assert np.array_equal(x.read(), a)
        _run(device, x, x, positions, _freq(pairs), pair_axis, neighbours, inverse, rotated, pos_dtype)  # in place, the same bits
        assert np.array_equal(x.read(), y.read())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
def test_packed_projection(device, dtype):
    """Queries and keys of a (B, S, 3, H, D) tensor in place, positions of their places: the values stay, and the inverse turns them back."""
    B, S, H, D = 3, 50, 2, 64
    a = round_to_dtype(normal(501, 0, (B, S, 3 * H, D)), dtype)
    buf, freq = AnyBuffer.from_numpy(device, a, dtype), AnyBuffer.from_numpy(device, _freq(D // 2), F32)
    st = i64s(S * 3 * H * D, 3 * H * D, D)
    turn = lambda inverse: device.lib.mg_rotary(buf.data_ptr(), buf.data_ptr(), None, freq.data_ptr(), None, B, S, 2 * H, D, D, st, st, None, 0, 0, 0, inverse,
                                                dtype, device.stream)
    turn(0)
    got = buf.to_numpy().reshape(a.shape)
    at = np.broadcast_to(np.arange(S), (1, B, S))
    _check(a[:, :, :2 * H], got[:, :, :2 * H], at, _freq(D // 2), [0] * (D // 2), False, False, dtype)
    assert np.array_equal(got[:, :, 2 * H:], a[:, :, 2 * H:])
    turn(1)
    back = buf.to_numpy().reshape(a.shape)[:, :, :2 * H]
    _check(got[:, :, :2 * H], back, at, _freq(D // 2), [0] * (D // 2), False, True, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
def test_far_and_shared_positions(device, dtype):
    """Positions up to 2^31 on either side, and positions that all sequences or all tokens share."""
    a = round_to_dtype(normal(502, 0, (2, 6, 2, 32)), dtype)
    f = _freq(16)
    far = np.array([[[0, 1, 2 ** 31 - 1, -2 ** 31, 123456789, -7]]])
    x, y = _View(device, a, dtype), _View(device, np.zeros_like(a), dtype)
    _run(device, x, y, far, f, None, 0, 0, 32, pos_strides=(0, 0, 1))
    _check(a, y.read(), np.broadcast_to(far, (1, 2, 6)), f, [0] * 16, False, False, dtype)
    one = np.array([[[5], [9]]])
    _run(device, x, y, one, f, None, 1, 0, 32, I64, pos_strides=(0, 1, 0))
    _check(a, y.read(), np.broadcast_to(one, (1, 2, 6)), f, [0] * 16, True, False, dtype)
    # a token that all positions share: x read with strides of 0
    B, S, H, D = a.shape
    first = AnyBuffer.from_numpy(device, a[0, 0], dtype)
    pos, freq = AnyBuffer.from_numpy(device, np.arange(B * S, dtype=np.int32)), AnyBuffer.from_numpy(device, f, F32)
    device.lib.mg_rotary(first.data_ptr(), y.ptr, pos.data_ptr(), freq.data_ptr(), None, B, S, H, D, 32, i64s(0, 0, D), i64s(*y.strides), i64s(0, S, 1), 1, I32, 0, 0,
                         dtype, device.stream)
    _check(np.broadcast_to(a[:1, :1], a.shape), y.read(), np.arange(B * S).reshape(1, B, S), f, [0] * 16, False, False, dtype)


@pytest.mark.gpu
def test_nothing_but_its_own_rows(device):
    """NaN and infinity stay in their pairs."""
    a = normal(503, 0, (1, 40, 3, 64)).astype(np.float32)
    x, y = _View(device, a, F32), _View(device, np.zeros_like(a), F32)
    _run(device, x, y, None, _freq(32), None, 0, 0, 64)
    want = y.read()
    bad = a.copy()
    bad[0, 7, 1, 5], bad[0, 9, 2, 40] = np.nan, np.inf
    x = _View(device, bad, F32)
    _run(device, x, y, None, _freq(32), None, 0, 0, 64)
    got = y.read()
    assert np.isnan(got[0, 7, 1, [5, 37]]).all() and not np.isfinite(got[0, 9, 2, [8, 40]]).any()
    for at in ((7, 1, 5), (7, 1, 37), (9, 2, 8), (9, 2, 40)):
        got[(0, *at)] = want[(0, *at)]
    assert np.array_equal(got, want)
