"""Gated layers' gradients with deferred sums recorded into HIP graphs, and the fp32 forward that keeps no projections.

Each graph is a step: both passes, the pending sums finished at its end.  It is replayed between eager steps on other inputs, with what the
pool hands out filled with NaN, and every replay gives the eager step's bits.
"""
import ctypes as C

import numpy as np
import pytest

from helpers import normal
from test_zz_recorded_scratch import _capture, _taken

pytestmark = pytest.mark.gpu

from mograd_amd import BF16, F16, F32, AnyBuffer  # noqa: E402
from mograd_amd.runtime import round_to_dtype  # noqa: E402


class _Step:
    def __init__(self, device, seed, M, F, K, dtype):
        self.device, self.shape, self.dtype, self.pending = device, (M, F, K), dtype, C.c_void_p()
        device.lib.mg_deferred_create(C.byref(self.pending))
        put = lambda i, shape, std=1.0: AnyBuffer.from_numpy(device, round_to_dtype(normal(seed, i, shape, std), dtype), dtype)
        self.x, self.w, self.bias, self.dy = put(0, (M, K)), put(1, (2 * F, K), K ** -0.5), put(2, 2 * F), put(3, (M, F))
        new = lambda n, t=dtype: AnyBuffer.create(t, device, n, fill=0.0)
        self.out = {"y": new(M * F), "alone": new(M * F), "gu": new(2 * M * F), "dx": new(M * K), "dw": new(2 * F * K, F32), "db": new(2 * F, F32),
                    "dw2": new(2 * F * K), "db2": new(2 * F)}

    def run(self, stream):
        lib, (M, F, K), t = self.device.lib, self.shape, self.dtype
        o, p = {n: b.data_ptr() for n, b in self.out.items()}, lambda b: b.data_ptr()
        lib.mg_gated_linear_fwd(p(self.x), p(self.w), p(self.bias), o["y"], o["gu"], M, F, K, 0, t, stream)
        lib.mg_gated_linear_fwd(p(self.x), p(self.w), p(self.bias), o["alone"], None, M, F, K, 0, t, stream)
        back = p(self.dy), o["gu"], p(self.x), p(self.w)
        lib.mg_gated_linear_bwd_deferred(*back, o["dx"], o["dw"], o["db"], M, F, K, 0, 0, t, F32, self.pending, stream)
        lib.mg_gated_linear_bwd_deferred(*back, None, o["dw2"], o["db2"], M, F, K, 0, 0, t, t, self.pending, stream)
        lib.mg_finish_deferred(self.pending, stream)

    def clear(self):
        for b in self.out.values():
            self.device.lib.mg_fill(b.data_ptr(), 5.0, b.numel, b.dtype, self.device.stream)

    def read(self):
        return {n: b.to_numpy() for n, b in self.out.items()}


# odd rows, which are copied; ranges of rows; fp32's plain product, which without kept projections takes scratch for them; its other one
CASES = [(BF16, 700, 101, 77, None), (F16, 2100, 96, 72, None), (BF16, 4096, 200, 384, None), (F32, 300, 90, 264, "64"), (F32, 1030, 140, 129, "128")]


@pytest.mark.parametrize("dtype,M,F,K,tile", CASES)
def test_graphs_keep_their_scratch(device, monkeypatch, dtype, M, F, K, tile):
    if not device.lib.mg_pool_enabled():
        pytest.skip("MOGRAD_POOL=0")
    if tile:
        monkeypatch.setenv("MOGRAD_HIP_GATED_TILE", tile)
        monkeypatch.setenv("MOGRAD_HIP_GATED_BWD_TILE", tile)
        monkeypatch.setenv("MOGRAD_HIP_GATED_SPLITS", "3")
    hip = C.CDLL("libamdhip64.so")
    steps, other = [_Step(device, 740 + i, M, F, K, dtype) for i in range(2)], _Step(device, 750, M, F, K, dtype)
    want = []
    for s in steps:
        s.run(device.stream)
        want.append(s.read())
        assert np.array_equal(want[-1]["alone"], want[-1]["y"])
    start = _taken(device)
    graphs = [_capture(hip, device, [s.run, s.run]) for s in steps]
    for _, _, grown in graphs:
        assert grown[0] > 0 and grown[1] == 0, "what a recorded step took stays taken, and serves the next one of its capture"
    sizes = (8, F, 2 * F, M, M * F // 2, M * F, 2 * M * F, F * K, 2 * F * K, 3 * 2 * F * K, 16 * 128 * 128)
    for turn in range(3):
        for s in steps:
            s.clear()
        filled = [AnyBuffer.create(F32, device, n, fill=float("nan")) for n in sizes for _ in range(2)]
        for _, exe, _ in graphs:
            other.run(device.stream)
            assert hip.hipGraphLaunch(exe, device.stream) == 0
            if turn == 1:
                device.synchronize()
            other.run(device.stream)
        for s, values in zip(steps, want):
            for n, v in s.read().items():
                assert np.array_equal(v, values[n]), (turn, n)
        assert all(np.isnan(b.to_numpy()).all() for b in filled), "a replay wrote into what the pool had given away"
        del filled
    for graph, exe, _ in graphs:
        assert hip.hipGraphExecDestroy(exe) == 0 and hip.hipGraphDestroy(graph) == 0
    device.synchronize()
    device.lib.mg_pool_free_recorded()
    assert _taken(device) <= start
    for s in steps + [other]:
        device.lib.mg_deferred_destroy(s.pending)
