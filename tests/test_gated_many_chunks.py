"""Gated layers whose odd rows are copied to chunks by more than one launch: 2^23 workgroups a launch, 2^24 + 1200 for these."""
import numpy as np
import pytest

from helpers import normal
from test_gated_large import _rows
from test_gated_linear import _check_forward

pytestmark = pytest.mark.gpu

from mograd_amd import BF16, AnyBuffer  # noqa: E402
from mograd_amd.runtime import round_to_dtype  # noqa: E402


def test_forward(device, monkeypatch):
    monkeypatch.setenv("MOGRAD_HIP_GATED_TILE", "128")  # (which copies)
    M, F, K = (1 << 23) + 600, 3, 4091
    device.lib.mg_pool_empty_cache()
    x = AnyBuffer.create(BF16, device, M * K, fill=0.25)  # 69 GB, and as much again for the copy
    w = AnyBuffer.from_numpy(device, wv := round_to_dtype(normal(810, 0, (2 * F, K), K ** -0.5), BF16), BF16)
    # rows at the ends of the launches and past 2^35 values; the others are all alike
    rows = np.array([0, 1, 4095, (1 << 22) - 1, 1 << 22, (1 << 22) + 1, (1 << 23) - 1, 1 << 23, M - 2, M - 1])
    values = round_to_dtype(normal(810, 1, (len(rows), K)), BF16)
    for r, v in zip(rows, values):
        device.lib.mg_copy_device(AnyBuffer(x.storage, BF16, K, int(r) * K).data_ptr(), AnyBuffer.from_numpy(device, v, BF16).data_ptr(), 2 * K, device.stream)
        device.synchronize()
    y, gu = AnyBuffer.create(BF16, device, M * F), AnyBuffer.create(BF16, device, M * 2 * F)
    device.lib.mg_gated_linear_fwd(x.data_ptr(), w.data_ptr(), None, y.data_ptr(), gu.data_ptr(), M, F, K, 0, BF16, device.stream)
    _check_forward({"x": values, "w": wv, "bias": None}, (_rows(y, rows, F), _rows(gu, rows, 2 * F)), BF16, "silu")
    same = np.setdiff1d(np.arange(M), rows)
    all_y, all_gu = y.to_numpy().reshape(M, F)[same], gu.to_numpy().reshape(M, 2 * F)[same]
    assert (all_y == all_y[0]).all() and (all_gu == all_gu[0]).all()
    _check_forward({"x": np.full((1, K), 0.25, np.float32), "w": wv, "bias": None}, (all_y[:1], all_gu[:1]), BF16, "silu")
    del x, y, gu
    device.synchronize()
    device.lib.mg_pool_empty_cache()
