"""fp32 gated layers: the error as a whole, and the range of the products of three bf16 numbers a value.

The 2-norm of a product's error.  An accumulator that n additions end loses at most a unit of its last place in each, 2^-23 of what it
holds then; from inputs of random signs that grows with the root of the additions, so the errors of one output add up to a root of the sum of
squares of 2^-23 sqrt(i / n), i = 1 .. n, of the final value's size: 2^-23 sqrt(n / 2).  fp32 instructions take 4 k, or 2, an addition: n = K / 2 at the
most.  The products of bf16 numbers take six additions for 16 k, n = 3 K / 8.  To that half a step of the result, and of each value that goes in.
Without the three products of second order the error would be 4.4e-6 whatever K is (first digits of a times the third ones of b, that of a's
third ones, and of the second ones: 2^-18 / sqrt(3) each of a's and b's rounding, and the like), and that is past every bound here.
"""
import numpy as np
import pytest

from oracle import oracle_np as O
from test_gated_linear import _backward, _forward, _inputs
from test_residual_norm import U

from mograd_amd import F32

SHAPES = [(150, 70, 264), (300, 90, 777), (130, 140, 4096)]


def _norm_bound(additions, values=1):
    return 2 * U * np.sqrt(additions / 2) + values * U


def _off(got, want):
    assert np.isfinite(got).all()
    return np.linalg.norm(got - want) / np.linalg.norm(want)


def _additions(tile, k):
    return 3 * k / 8 if tile in ("128", "256") else k / 2


def _three(a):
    a = a.astype(np.float32)
    parts = []
    for _ in range(3):
        bits = a.view(np.uint32).astype(np.uint64)
        head = ((bits + 0x7fff + ((bits >> 16) & 1)) & 0xffff0000).astype(np.uint32).view(np.float32)
        parts.append(head.astype(np.float64))
        a = (a - head).astype(np.float32)
    return parts


@pytest.mark.parametrize("M,F,K", SHAPES)
def test_bounds_see_the_products_of_second_order(M, F, K):
    """What is left out of the nine products is far below the bounds, the next three are not."""
    p = _inputs(434, M, F, K, F32, bias=False)
    a, b = _three(p["x"]), _three(p["w"])
    want = p["x"].astype(np.float64) @ p["w"].astype(np.float64).T
    first = a[0] @ b[0].T + (a[0] @ b[1].T + a[1] @ b[0].T)
    six = first + (a[0] @ b[2].T + a[1] @ b[1].T + a[2] @ b[0].T)
    bound = _norm_bound(_additions("128", K))
    assert _off(six, want) <= 0.05 * bound and _off(first, want) > bound


@pytest.mark.gpu
@pytest.mark.parametrize("M,F,K", SHAPES)
@pytest.mark.parametrize("tile", ["16", "64", "128", "256"])
def test_forward(device, monkeypatch, tile, M, F, K):
    monkeypatch.setenv("MOGRAD_HIP_GATED_TILE", tile)
    for offset in (0, 1):
        p = _inputs(434, M, F, K, F32, bias=False)
        _, gu = _forward(device, p, F32, "silu", offset=offset)
        _, want = O.gated_linear_fwd(p["x"], p["w"], None, "silu")
        off = _off(gu, want)
        print(f"forward {tile} K={K}: {off:.3g} of {_norm_bound(_additions(tile, K)):.3g}")
        assert off <= _norm_bound(_additions(tile, K)), off


@pytest.mark.gpu
@pytest.mark.parametrize("M,F,K", [(264, 150, 140), (777, 200, 90), (4096, 390, 130)])
@pytest.mark.parametrize("tile,splits", [("64", "1"), ("128", "1"), ("128", "3"), ("256", "1")])
def test_backward(device, monkeypatch, tile, splits, M, F, K):
    """max(g, 0): dg and du are products of two or three values, an error of 2^-24 a product in what the matrix instructions take."""
    monkeypatch.setenv("MOGRAD_HIP_GATED_BWD_TILE", tile)
    monkeypatch.setenv("MOGRAD_HIP_GATED_SPLITS", splits)
    p = _inputs(435, M, F, K, F32)
    got = _backward(device, p, F32, F32, "relu")
    dx, dw, _, _ = O.gated_linear_bwd(p["dy"], p["gu"], p["x"], p["w"], "relu")
    for n, want, k in (("dx", dx, 2 * F), ("dw", dw, M)):
        off, bound = _off(got[n], want), _norm_bound(_additions(tile, k), 3)
        print(f"backward {n} {tile} k={k}: {off:.3g} of {bound:.3g}")
        assert off <= bound, (n, off)


# Three bf16 numbers hold fp32's last digit, down to 2^-133, in numbers from 2^-110 on; the weights here are 2^-4 in the mean.
@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** -104, 2.0 ** -83, 2.0 ** 50, 2.0 ** 104])
@pytest.mark.parametrize("tile", ["128", "256"])
def test_far_from_one(device, monkeypatch, tile, size):
    """Values far from 1 in one operand, in the other what brings the products back."""
    monkeypatch.setenv("MOGRAD_HIP_GATED_TILE", tile)
    monkeypatch.setenv("MOGRAD_HIP_GATED_BWD_TILE", tile)
    M, F, K = 300, 150, 264
    p = _inputs(436, M, F, K, F32, bias=False)
    q = {**p, "x": (p["x"] * np.float32(size)).astype(np.float32), "w": (p["w"] / np.float32(size)).astype(np.float32)}
    _, gu = _forward(device, q, F32, "silu")
    want = O.gated_linear_fwd(p["x"], p["w"], None, "silu")[1]  # (a power of two: the same digits)
    off = _off(gu, want)
    print(f"forward {tile}: {off:.3g}")
    assert off <= _norm_bound(_additions(tile, K)), off
    got = _backward(device, q, F32, F32, "relu")
    dx, dw, _, _ = O.gated_linear_bwd(p["dy"], p["gu"], p["x"], p["w"], "relu")
    for n, ref, k, back in (("dx", dx, 2 * F, 1 / size), ("dw", dw, M, size)):
        off = _off(got[n].astype(np.float64) / back, ref)
        print(f"backward {n} {tile}: {off:.3g}")
        assert off <= _norm_bound(_additions(tile, k), 3), (n, off)


@pytest.mark.gpu
@pytest.mark.parametrize("tile", ["128", "256"])
def test_infinities_stay_where_they_are(device, monkeypatch, tile):
    """An infinity, or a number that bf16 rounds to one, makes NaN of the outputs that it is in, and of no others; 3.39e38 is a number."""
    monkeypatch.setenv("MOGRAD_HIP_GATED_TILE", tile)
    monkeypatch.setenv("MOGRAD_HIP_GATED_BWD_TILE", tile)
    M, F, K = 300, 70, 100
    p = _inputs(437, M, F, K, F32)
    y, gu = _forward(device, p, F32, "silu")
    grads = _backward(device, p, F32, F32, "silu")
    for bad in (np.inf, -np.inf, np.nan, np.float32(3.3965e38)):
        q = {k: v.copy() for k, v in p.items()}
        q["x"][[5, 290], [3, 99]] = bad
        y2, gu2 = _forward(device, q, F32, "silu")
        rest = np.setdiff1d(np.arange(M), [5, 290])
        assert np.isnan(y2[[5, 290]]).all() and np.isnan(gu2[[5, 290]]).all()
        assert np.array_equal(y2[rest], y[rest]) and np.array_equal(gu2[rest], gu[rest])
        got = _backward(device, q, F32, F32, "silu")
        rest = np.setdiff1d(np.arange(K), [3, 99])
        assert np.isnan(got["dw"][:, [3, 99]]).all() and np.array_equal(got["dw"][:, rest], grads["dw"][:, rest])
        assert np.array_equal(got["dx"], grads["dx"]) and np.array_equal(got["db"], grads["db"])
        q = {k: v.copy() for k, v in p.items()}
        q["w"][[7, F + 60], [98, 0]] = bad
        y2, gu2 = _forward(device, q, F32, "silu")
        assert np.isnan(gu2[:, [7, F + 60]]).all() and np.isnan(y2[:, [7, 60]]).all()
        rest = np.setdiff1d(np.arange(F), [7, 60])
        assert np.array_equal(y2[:, rest], y[:, rest])
        got = _backward(device, q, F32, F32, "silu")
        rest = np.setdiff1d(np.arange(K), [0, 98])
        assert np.isnan(got["dx"][:, [0, 98]]).all() and np.array_equal(got["dx"][:, rest], grads["dx"][:, rest])
        assert np.array_equal(got["dw"], grads["dw"])
    q = {k: v.copy() for k, v in p.items()}
    q["x"][5, 3], q["w"][:, 3] = np.float32(3.39e38), np.float32(2.0 ** -126)
    _, gu2 = _forward(device, q, F32, "silu")
    want = O.gated_linear_fwd(q["x"], q["w"], q["bias"], "silu")[1]
    mass = np.abs(q["x"]).astype(np.float64) @ np.abs(q["w"]).astype(np.float64).T + np.abs(q["bias"])
    assert (np.abs(gu2 - want) <= (K + 17) * U * mass).all()
