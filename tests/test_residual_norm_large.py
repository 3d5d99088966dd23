"""The residual norm at the sizes that only large tensors reach; tolerances and helpers of tests/test_residual_norm.py."""
import numpy as np
import pytest

from helpers import normal
from test_residual_norm import _backward, _check_backward, _check_forward, _check_kept, _forward, _inputs, _saved

from mograd_amd import BF16, F16, F32
from mograd_amd.runtime import round_to_dtype

pytestmark = pytest.mark.gpu


# rows, cols, gates: rows of fewer columns than a chunk, more of them than the launch has workgroups, and than 2^32 threads would take at
# a workgroup each
@pytest.mark.parametrize("dtype,rows,cols,gates,post,pre", [(BF16, 70001, 7, 1, 1, 1), (F16, 131074, 3, 2, 0, 1), (F32, 70002, 3, 3, 1, 0),
                                                            (BF16, 4194312, 3, 8, 1, 1)])
def test_more_narrow_rows_than_workgroups(device, dtype, rows, cols, gates, post, pre):
    p = _inputs(41, rows, cols, gates, post, pre, dtype)
    got = _forward(device, p, dtype, 0.75, keep8=True)
    _check_forward(p, got, dtype, 0.75)
    _check_kept(p, got, dtype)
    saved = _saved(p, dtype, 1.25)
    _check_backward(p, saved, _backward(device, p, saved, dtype, F32, 1.25), dtype, F32, 1.25)


def test_second_stage_of_more_columns_than_a_launch_has(device):
    """One row of 2^25 + 33 columns: the sums over the rows are the row's own values, each in its column."""
    cols = (1 << 25) + 33
    a = round_to_dtype(normal(42, 0, (1, cols)), BF16)
    one = np.ones(1, np.float32)
    p = {"f": a, "gate": np.full((1, cols), 0.5, np.float32), "post": None, "pre": (np.ones(cols, np.float32),) * 2, "dx": a[:, ::-1], "dh_out": a}
    got = _backward(device, p, {"h_out": a, "pre_mean": 0 * one, "pre_rstd": one, "post_mean": None, "post_rstd": None}, BF16, F32, 1.0)
    assert np.array_equal(got["dpre_beta"], a[0, ::-1])
    assert np.array_equal(got["dpre_gamma"], a[0] * a[0, ::-1])  # (a product of two bf16 numbers is one of fp32)
    # dgate = d f in fp32, df = d / 2 rounded to bf16: off by at most 2^-8 / (1 - 2^-8) of itself
    want = 2 * got["df"].astype(np.float64) * a
    assert (np.abs(got["dgate"] - want) <= 1.01 * 2.0 ** -8 * np.abs(want)).all()


# rows, cols, gates: more rows than the forward's workgroups take at once, so that a row's place goes on to others and their gate rows,
# in every layout that so many rows have (16 lanes to 256 threads with two chunks each); gate rows end anywhere in a step
FORWARD = [(F16, 40000, 64, 32), (BF16, 33000, 250, 8), (BF16, 17003, 384, 7), (BF16, 9009, 1000, 13), (F16, 8200, 2040, 41), (BF16, 8200, 4096, 41),
           (F32, 36000, 30, 9), (F32, 9009, 500, 1001), (F32, 8200, 1020, 0), (F32, 8200, 1400, 25)]


@pytest.mark.parametrize("dtype,rows,cols,gates", FORWARD)
def test_forward_of_many_rows(device, dtype, rows, cols, gates):
    p = _inputs(43, rows, cols, gates, 1, 1, dtype)
    for kw in (dict(), dict(offset=1, in_place=True)):
        got = _forward(device, p, dtype, 0.75, keep8=True, **kw)
        _check_forward(p, got, dtype, 0.75)
        _check_kept(p, got, dtype)


@pytest.mark.parametrize("post,pre", [(0, 1), (1, 0), (0, 0)])
@pytest.mark.parametrize("dtype,rows,cols,gates", [(BF16, 9009, 1000, 13), (F16, 8200, 2040, 41), (F32, 8200, 1400, 25)])
def test_forward_of_many_rows_without_a_norm(device, dtype, rows, cols, gates, post, pre):
    p = _inputs(44, rows, cols, gates, post, pre, dtype)
    for kw in (dict(in_place=True), dict(offset=1)):
        _check_forward(p, _forward(device, p, dtype, 0.75, **kw), dtype, 0.75)


# 16 MiB and more, where the pieces of a gate row lie row by row between each other: every layout, one gate row, several, and of odd lengths;
# both types of the gradients
BACKWARD = [(BF16, BF16, 140000, 64, 7), (F16, F32, 33000, 256, 8), (BF16, F32, 22100, 384, 13), (F16, F16, 22101, 384, 1),
            (BF16, BF16, 9009, 1000, 1), (F16, F32, 9009, 1000, 13), (F16, F32, 8200, 2040, 41), (BF16, BF16, 2190, 4096, 3),
            (F32, F32, 2050, 4096, 5), (BF16, BF16, 1030, 16384, 2), (F32, F32, 40001, 120, 1)]


@pytest.mark.parametrize("dtype,grads,rows,cols,gates", BACKWARD)
def test_backward_of_large_tensors(device, dtype, grads, rows, cols, gates):
    p = _inputs(45, rows, cols, gates, 1, 1, dtype)
    saved = _saved(p, dtype, 1.25)
    for kw, run in ((dict(), dict(in_place=True)), (dict(act8=True), dict(offset=1))):
        got = _backward(device, p, saved, dtype, grads, 1.25, **kw, **run)
        _check_backward(p, saved, got, dtype, grads, 1.25, **kw)


@pytest.mark.parametrize("dtype,grads", [(BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("rows,cols,gates", [(6, 3, 2), (67, 130, 1), (40, 384, 4), (24, 1001, 3), (6, 4100, 0), (3, 20001, 3), (2600, 40, 1300)])
@pytest.mark.parametrize("post,pre", [(1, 1), (0, 1), (1, 0)])
def test_backward_in_the_other_type_of_gradients(device, dtype, grads, rows, cols, gates, post, pre):
    p = _inputs(46, rows, cols, gates, post, pre, dtype)
    saved = _saved(p, dtype, 1.25)
    for kw, run in ((dict(), dict()), (dict(act8=True), dict(offset=1))):
        got = _backward(device, p, saved, dtype, grads, 1.25, **kw, **run)
        _check_backward(p, saved, got, dtype, grads, 1.25, **kw)
