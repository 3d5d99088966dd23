"""The residual norm at the sizes that only large tensors reach; tolerances and helpers of tests/test_residual_norm.py."""
import pytest

from test_residual_norm import _backward, _check_backward, _check_forward, _check_kept, _forward, _inputs, _saved

from mograd_amd import BF16, F16, F32

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
