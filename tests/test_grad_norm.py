"""The global norm of gradients, gradients scaled down to a largest norm, and optimizer steps from them.

Tolerances: the norm is a sum in 64 bits rounded once to fp32, 2^-24 of it (2^-23 with room for the 64-bit sums); a clipped value takes
the norm's rounding, one of the quotient and one of the product, 4 x 2^-24 with room, and half a step of its own type.
"""
import ctypes as C

import numpy as np
import pytest

from helpers import normal
from oracle import oracle_np as O
from test_residual_norm import FLOATS, U, _close, _half_step

import mograd_amd
from mograd_amd import BF16, F16, F32, I32, AnyBuffer, MogradError
from mograd_amd.runtime import round_to_dtype


def _arrays(pointers, numels, dtypes):
    n = len(pointers)
    return (C.c_void_p * n)(*pointers), (C.c_int64 * n)(*numels), (C.c_int * n)(*dtypes)


def test_refusals():
    """Answered before anything is launched; the pointers are never followed."""
    lib = mograd_amd.load()
    p = 4096

    def call(pointers=(p, p), out=(p, 2 * p), numels=(5, 6), dtypes=(F32, BF16), count=2, max_norm=1.0, norm=p, clip=True):
        g, n, t = _arrays(pointers, numels, dtypes)
        if clip:
            return lib.mg_clip_grads(g, (C.c_void_p * 2)(*out) if out else None, n, t, count, max_norm, norm, None)
        return lib.mg_grad_norm(g, n, t, count, norm, None)

    both = [dict(count=-1), dict(numels=(5, -1)), dict(numels=(5, 1 << 50)), dict(dtypes=(F32, I32)), dict(dtypes=(9, F32)), dict(pointers=(p, None))]
    for bad in both + [dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(out=None), dict(out=(None, p)), dict(out=(p, p))]:
        with pytest.raises(MogradError) as e:
            call(**bad)
        assert e.value.status == 1 and "clip_grads" in str(e.value), bad
    for bad in both + [dict(norm=None)]:
        with pytest.raises(MogradError) as e:
            call(clip=False, **bad)
        assert e.value.status == 1 and "grad_norm" in str(e.value), bad
    for fn, args in ((lib.mg_grad_norm, (None, None, None, 1, p, None)), (lib.mg_clip_grads, (None, None, None, None, 1, 1.0, p, None))):
        with pytest.raises(MogradError):
            fn(*args)
    q = C.c_void_p(p)
    for bad in (dict(norm=None), dict(most=-1.0), dict(most=float("nan"))):
        norm, most = bad.get("norm", q), bad.get("most", 1.0)
        with pytest.raises(MogradError) as e:
            lib.mg_adam_step_clipped(q, q, q, q, 4, 0.1, 0.9, 0.99, 1e-8, 0.0, 1, 0, norm, most, None)
        assert e.value.status == 1
        with pytest.raises(MogradError) as e:
            lib.mg_sgd_step_clipped(q, q, 4, 0.1, norm, most, None)
        assert e.value.status == 1
    for bad in (dict(n=-1), dict(t=0)):
        with pytest.raises(MogradError):
            lib.mg_adam_step_clipped(q, q, q, q, bad.get("n", 4), 0.1, 0.9, 0.99, 1e-8, 0.0, bad.get("t", 1), 0, q, 1.0, None)


# ---- on the GPU ----------------------------------------------------------------------------


class _Tensors:
    """Arrays on the device, tensor i `i % 4` elements into a buffer of its own, with guards around what is written."""

    def __init__(self, device, arrays, dtypes):
        self.device, self.dtypes, self.sizes = device, list(dtypes), [a.size for a in arrays]
        self.at = [i % 4 for i in range(len(arrays))]
        self.bufs = [AnyBuffer.from_numpy(device, np.concatenate([np.full(k, -3.0, np.float32), a, np.full(5, -3.0, np.float32)]), t)
                     for a, t, k in zip(arrays, dtypes, self.at)]

    def pointers(self):
        return [AnyBuffer(b.storage, t, n, k).data_ptr().value if n else None for b, t, n, k in zip(self.bufs, self.dtypes, self.sizes, self.at)]

    def read(self):
        out = []
        for b, n, k in zip(self.bufs, self.sizes, self.at):
            v = b.to_numpy()
            assert (v[:k] == -3).all() and (v[k + n:] == -3).all(), "written outside"
            out.append(v[k:k + n])
        return out


def _clip(device, arrays, dtypes, max_norm, in_place=False):
    g = _Tensors(device, arrays, dtypes)
    out = g if in_place else _Tensors(device, [np.full_like(a, 7.0) for a in arrays], dtypes)
    norm = AnyBuffer.create(F32, device, 1, fill=-1.0)
    p, n, t = _arrays(g.pointers(), g.sizes, dtypes)
    o = (C.c_void_p * len(arrays))(*out.pointers())
    device.lib.mg_clip_grads(p, o, n, t, len(arrays), max_norm, norm.data_ptr(), device.stream)
    clipped, got = out.read(), norm.to_numpy()[0]
    if not in_place:
        norm2 = AnyBuffer.create(F32, device, 1, fill=-1.0)
        device.lib.mg_grad_norm(p, n, t, len(arrays), norm2.data_ptr(), device.stream)
        assert norm2.to_numpy()[0] == got or np.isnan(got)
        for a, b in zip(g.read(), arrays):
            assert np.array_equal(a, b, equal_nan=True)
    return got, clipped


def _gradients(seed, sizes, dtypes, std=0.02):
    return [round_to_dtype(normal(seed, i, n, std * (1 + i % 3)), t) for i, (n, t) in enumerate(zip(sizes, dtypes))]


# one element, none, a chunk and one over, a piece and one over, many tensors (more than one launch's), one long one
SIZES = [[1], [0, 3, 0], [8, 9, 7, 64], [2048, 2049, 2047, 1], [5000, 1, 0, 70001, 333], [1 + i * 37 % 500 for i in range(300)], [300, 3000001]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [*FLOATS, None])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
def test_against_float64(device, sizes, dtype):
    dtypes = [dtype if dtype is not None else FLOATS[i % 3] for i in range(len(sizes))]
    g = _gradients(600, sizes, dtypes)
    norm = O.grad_norm(g)
    for share in (0.0, 0.3, 0.999, 1.001, np.inf):
        want_norm, want = O.clip_grads(g, norm * share)
        for in_place in (False, True):
            got_norm, got = _clip(device, g, dtypes, norm * share, in_place)
            assert abs(got_norm - want_norm) <= 2 * U * want_norm
            for v, w, a, t in zip(got, want, g, dtypes):
                _close(v, w, _half_step(w, t) + 4 * U * np.abs(w), "clipped")
                if share > 1:
                    assert np.array_equal(v, a)


@pytest.mark.gpu
def test_values_whose_squares_leave_fp32(device):
    for size in (1e-30, 1e25):
        g = [np.full(10000, size, np.float32), np.full(77, -size, np.float32)]
        norm, got = _clip(device, g, [F32, F32], size)
        want, clipped = O.clip_grads(g, size)
        assert abs(norm - want) <= 2 * U * want
        _close(got[0], clipped[0], 5 * U * np.abs(clipped[0]), "clipped")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
def test_norms_that_are_no_numbers(device, dtype):
    """NaN: the gradients stay as they are.  Infinite: zeros, and NaN where a gradient is infinite.  Zero: zeros."""
    g = _gradients(601, [5000, 300], [dtype, dtype])
    g[1][7] = np.nan
    norm, got = _clip(device, g, [dtype, dtype], 0.5)
    assert np.isnan(norm) and all(np.array_equal(a, b, equal_nan=True) for a, b in zip(got, g))
    g[1][7] = np.inf
    norm, got = _clip(device, g, [dtype, dtype], 0.5)
    assert norm == np.inf and np.isnan(got[1][7])
    got[1][7] = 0
    assert all((v == 0).all() for v in got)
    zero = [np.zeros(3000, np.float32)]
    norm, got = _clip(device, zero, [dtype], 0.0)
    assert norm == 0 and (got[0] == 0).all()


@pytest.mark.gpu
def test_no_tensors(device):
    norm = AnyBuffer.create(F32, device, 1, fill=5.0)
    device.lib.mg_grad_norm(None, None, None, 0, norm.data_ptr(), device.stream)
    assert norm.to_numpy()[0] == 0
    p, n, t = _arrays([None], [0], [F16])
    norm = AnyBuffer.create(F32, device, 1, fill=5.0)
    device.lib.mg_clip_grads(p, p, n, t, 1, 1.0, norm.data_ptr(), device.stream)
    assert norm.to_numpy()[0] == 0


@pytest.mark.gpu
def test_without_a_place_for_the_norm(device):
    g = _gradients(602, [4000], [F32])
    buf = AnyBuffer.from_numpy(device, g[0], F32)
    p, n, t = _arrays([buf.data_ptr().value], [4000], [F32])
    device.lib.mg_clip_grads(p, p, n, t, 1, 0.1, None, device.stream)
    want = O.clip_grads(g, 0.1)[1][0]
    _close(buf.to_numpy(), want, 5 * U * np.abs(want), "clipped")


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 5, 1024, 100003])
@pytest.mark.parametrize("share", [0.25, 2.0])
def test_optimizer_steps_from_clipped_gradients(device, n, share):
    """Bit for bit the plain steps from gradients that mg_clip_grads has scaled; the gradients stay as they were."""
    w, g, m = (normal(603, i, n, s).astype(np.float32) for i, s in ((0, 1.0), (1, 0.1), (2, 0.01)))
    v = np.square(normal(603, 3, n, 0.1)).astype(np.float32)
    lib, s = device.lib, device.stream
    put = lambda a: AnyBuffer.from_numpy(device, a, F32)
    grads, norm = put(g), AnyBuffer.create(F32, device, 1)
    most = float(np.float32(share * O.grad_norm([g])))
    p, k, t = _arrays([grads.data_ptr().value], [n], [F32])
    clipped = AnyBuffer.create(F32, device, n)
    o = (C.c_void_p * 1)(clipped.data_ptr().value)
    lib.mg_clip_grads(p, o, k, t, 1, most, norm.data_ptr(), s)
    hyper = (1e-2, 0.9, 0.999, 1e-8)
    for decay, decoupled in ((0.0, 0), (0.1, 0), (0.1, 1)):
        a, b = [put(x) for x in (w, m, v)], [put(x) for x in (w, m, v)]
        lib.mg_adam_step_clipped(a[0].data_ptr(), grads.data_ptr(), a[1].data_ptr(), a[2].data_ptr(), n, *hyper, decay, 3, decoupled, norm.data_ptr(), most, s)
        lib.mg_adam_step(b[0].data_ptr(), clipped.data_ptr(), b[1].data_ptr(), b[2].data_ptr(), n, *hyper, decay, 3, decoupled, s)
        for x, y in zip(a, b):
            assert np.array_equal(x.to_numpy(), y.to_numpy())
    a, b = put(w), put(w)
    lib.mg_sgd_step_clipped(a.data_ptr(), grads.data_ptr(), n, 0.1, norm.data_ptr(), most, s)
    lib.mg_sgd_step(b.data_ptr(), clipped.data_ptr(), n, 0.1, s)
    assert np.array_equal(a.to_numpy(), b.to_numpy()) and np.array_equal(grads.to_numpy(), g)
    assert (a.to_numpy() != put(w).to_numpy()).any()


@pytest.mark.gpu
def test_twice_gives_the_same_bits(device):
    g = _gradients(604, [100000, 33, 4096], [F32, BF16, F16])
    a, b = (_clip(device, g, [F32, BF16, F16], 0.7) for _ in range(2))
    assert a[0] == b[0] and all(np.array_equal(x, y) for x, y in zip(a[1], b[1]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_thousands_of_small_tensors(device, dtype):
    """More pieces than each workgroup adds up for itself; the tensors lie in one array, without gaps."""
    sizes = [i % 6 for i in range(10001)]
    g = _gradients(605, sizes, [dtype] * len(sizes))
    flat = np.concatenate(g)
    start = np.cumsum([0] + sizes)
    buf, out = AnyBuffer.from_numpy(device, flat, dtype), AnyBuffer.create(dtype, device, flat.size, fill=7.0)
    norm, norm2 = (AnyBuffer.create(F32, device, 1, fill=-1.0) for _ in range(2))
    at = lambda b: [AnyBuffer(b.storage, dtype, n, int(k)).data_ptr().value if n else None for n, k in zip(sizes, start)]
    want_norm, want = O.clip_grads(g, O.grad_norm(g) * 0.4)
    p, n, t = _arrays(at(buf), sizes, [dtype] * len(sizes))
    most = float(O.grad_norm(g) * 0.4)
    device.lib.mg_clip_grads(p, (C.c_void_p * len(sizes))(*at(out)), n, t, len(sizes), most, norm.data_ptr(), device.stream)
    device.lib.mg_grad_norm(p, n, t, len(sizes), norm2.data_ptr(), device.stream)
    assert norm.to_numpy()[0] == norm2.to_numpy()[0]
    assert abs(norm.to_numpy()[0] - want_norm) <= 2 * U * want_norm
    w = np.concatenate(want)
    _close(out.to_numpy(), w, _half_step(w, dtype) + 4 * U * np.abs(w), "clipped")
    assert np.array_equal(buf.to_numpy(), flat)
