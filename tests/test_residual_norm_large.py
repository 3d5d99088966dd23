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
