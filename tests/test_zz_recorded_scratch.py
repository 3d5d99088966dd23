"""What recorded calls of mg_residual_norm_bwd and mg_linear_bwd_act8 take from the pool: shared by the calls of one stream in one
capture, kept from everyone else, and given back by mg_pool_free_recorded."""
import ctypes as C

import numpy as np
import pytest

from test_zz_act8_graphs import _Work

pytestmark = pytest.mark.gpu

from mograd_amd import BF16, F32, AnyBuffer  # noqa: E402
from mograd_amd._lib import PoolStats  # noqa: E402


def _taken(device):
    stats = PoolStats()
    device.lib.mg_pool_get_stats(stats)
    return stats.allocated_bytes


def _capture(hip, device, runs):
    graph, exe, grown = C.c_void_p(), C.c_void_p(), []
    assert hip.hipStreamBeginCapture(device.stream, C.c_int(0)) == 0
    try:
        for run in runs:
            before = _taken(device)
            run(device.stream)
            grown.append(_taken(device) - before)
    finally:
        assert hip.hipStreamEndCapture(device.stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)) == 0
    return graph, exe, grown


@pytest.mark.parametrize("dtype,route", [(BF16, "1"), (F32, "1"), (F32, "0")])
def test_scratch_of_a_capture(device, monkeypatch, dtype, route):
    if not device.lib.mg_pool_enabled():
        pytest.skip("MOGRAD_POOL=0")
    monkeypatch.setenv("MOGRAD_HIP_ACT8_ROUTE", route)
    hip = C.CDLL("libamdhip64.so")
    works = [_Work(device, 340 + i, 700, 96, 72, dtype) for i in range(3)]
    want = []
    for w in works:
        w.run(device.stream)
        want.append(w.read())
    start = _taken(device)
    first, second = (_capture(hip, device, [w.run for w in works]) for _ in range(2))
    for _, _, grown in (first, second):
        assert grown[0] > 0 and grown[1:] == [0, 0]
    held = _taken(device)
    assert held == start + first[2][0] + second[2][0]
    for turn in range(3):
        for graph, exe, _ in (first, second):
            for w in works:
                w.clear()
            filled = [AnyBuffer.create(F32, device, n, fill=float("nan")) for n in (96, 700, 700 * 96, 40 * 96, 128 * 128, 16 * 128 * 128)]
            assert hip.hipGraphLaunch(exe, device.stream) == 0
            if turn == 1:
                device.synchronize()
            for w, values in zip(works, want):
                for n, v in w.read().items():
                    assert np.array_equal(v, values[n]), (turn, n)
            del filled
            works[turn].run(device.stream)  # an eager call between the replays
    assert _taken(device) == held
    for graph, exe, _ in (first, second):
        assert hip.hipGraphExecDestroy(exe) == 0 and hip.hipGraphDestroy(graph) == 0
    device.synchronize()
    device.lib.mg_pool_free_recorded()
    assert _taken(device) <= start  # (what other tests' graphs left goes back with it)
