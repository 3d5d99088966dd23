"""Gated Linear layers whose projections are infinite: what the gates' formulas give there, from every kernel.

sigmoid(g) is 1 and 0 there and max(g, 0) infinite and 0; g sigmoid(g) and g Phi(g) are infinite, and at -infinity a product of infinity
and 0, NaN.  The other factor is 1/2 and exact, so nothing is rounded; the columns between keep the bounds of finite ones.
"""
import numpy as np
import pytest

from test_gated_linear import GATES, WAYS, _backward, _check_forward, _forward, _inputs
from test_residual_norm import FLOATS

from mograd_amd import F32

pytestmark = pytest.mark.gpu

INF = np.inf
ACT = {"silu": (INF, np.nan), "gelu": (INF, np.nan), "gelu_tanh": (INF, np.nan), "sigmoid": (1.0, 0.0), "relu": (INF, 0.0)}


def _with_infinities(seed, M, F, K, dtype):
    p = _inputs(seed, M, F, K, dtype)
    up, down = np.arange(0, F, 7), np.arange(1, F, 7)
    p["bias"][up], p["bias"][down] = INF, -INF
    for at in (up, down):
        p["w"][F + at], p["bias"][F + at] = 0, 0.5
    return p, up, down, np.setdiff1d(np.arange(F), np.concatenate([up, down]))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("M,F,K", [(5, 24, 40), (130, 72, 65)])
@pytest.mark.parametrize("gate", GATES)
def test_forward(device, monkeypatch, gate, M, F, K, dtype):
    p, up, down, rest = _with_infinities(450, M, F, K, dtype)
    finite = {**p, "w": p["w"][np.concatenate([rest, F + rest])], "bias": p["bias"][np.concatenate([rest, F + rest])]}
    for tile, splits in [(None, None)] + WAYS:
        if tile:
            monkeypatch.setenv("MOGRAD_HIP_GATED_TILE", tile)
            monkeypatch.setenv("MOGRAD_HIP_GATED_SPLITS", splits)
        for offset in (0, 1):
            y, gu = _forward(device, p, dtype, gate, offset=offset)
            for at, g, act in ((up, INF, ACT[gate][0]), (down, -INF, ACT[gate][1])):
                assert (gu[:, at] == g).all() and (gu[:, F + at] == 0.5).all(), (tile, offset)
                assert np.array_equal(y[:, at], np.full((M, len(at)), 0.5 * act, np.float32), equal_nan=True), (tile, offset, y[0, at])
            _check_forward(finite, (y[:, rest], gu[:, np.concatenate([rest, F + rest])]), dtype, gate)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("gate", ["sigmoid", "relu"])
def test_backward(device, monkeypatch, gate, dtype):
    """A gate closed or wide open for good: act'(g) is 0 at -infinity, for sigmoid at infinity too, and du = dy act(g)."""
    M, F, K = 70, 24, 40
    p = _inputs(451, M, F, K, dtype)
    closed, wide = np.arange(0, F, 5), np.arange(1, F, 5)
    p["gu"][:, closed] = -INF
    if gate == "sigmoid":
        p["gu"][:, wide] = INF
    p["gu"][:, F:] = 0.5
    p["dy"][:] = 0.25
    p["x"][:] = 0.5
    for tile in ("64", "128", "256") if dtype == F32 else ("0",):
        if dtype == F32:
            monkeypatch.setenv("MOGRAD_HIP_GATED_BWD_TILE", tile)
        got = _backward(device, p, dtype, F32, gate)
        # 70 rows of dy 1/4: sums of at most 17.5, exact in fp32 in any order; dw of x 1/2
        assert (got["db"][closed] == 0).all() and (got["db"][F + closed] == 0).all()
        assert (got["dw"][closed] == 0).all() and (got["dw"][F + closed] == 0).all()
        if gate == "sigmoid":
            assert (got["db"][wide] == 0).all() and (got["db"][F + wide] == 17.5).all()
            assert (got["dw"][wide] == 0).all() and (got["dw"][F + wide] == 8.75).all()
        assert np.isfinite(got["dx"]).all()
