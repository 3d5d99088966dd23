"""mg_residual_norm_bwd and mg_linear_bwd_act8, which take scratch, recorded into HIP graphs: what a recorded call took stays its
own, so that two graphs and the program's eager calls, which take scratch of the same sizes, do not write into each other's.

Each graph holds the forward, a block's pair of gradients and a Linear layer's; it is replayed with eager calls on other inputs,
allocations that fill what the pool hands out, and synchronizations in between, and every replay gives the eager call's bits.
"""
import ctypes as C

import numpy as np
import pytest

from helpers import normal

pytestmark = pytest.mark.gpu

from mograd_amd import BF16, F32, I32, AnyBuffer  # noqa: E402
from mograd_amd._lib import PoolStats  # noqa: E402
from mograd_amd.runtime import round_to_dtype  # noqa: E402


class _Work:
    """One block's operators on inputs of a seed, with buffers of its own."""

    def __init__(self, device, seed, rows, cols, width, dtype):
        self.device, self.shape, self.dtype = device, (rows, cols, width), dtype
        put = lambda i, shape, std=1.0, mean=0.0: AnyBuffer.from_numpy(device, round_to_dtype(normal(seed, i, shape, std, mean), dtype), dtype)
        self.f, self.h, self.dx, self.dh_out = (put(i, (rows, cols)) for i in range(4))
        self.gate, self.pg, self.pb, self.ng, self.nb = (put(10 + i, cols, 0.2, 1.0) for i in range(5))
        self.dy, self.w = put(20, (rows, width), 0.1), put(21, (width, cols), 0.1)
        new = lambda n, t=dtype: AnyBuffer.create(t, device, n, fill=0.0)
        self.out = {"h_out": new(rows * cols), "x": new(rows * cols), "df": new(rows * cols), "dh": new(rows * cols), "dx": new(rows * cols),
                    "dw": new(width * cols, F32), "db": new(width, F32)}
        for n in ("dgate", "dpg", "dpb", "dng", "dnb"):
            self.out[n] = new(cols, F32)
        self.stats = [new(rows, F32) for _ in range(4)]
        words = -(-device.lib.mg_act8_bytes(rows, cols) // 4)
        self.f8, self.x8 = new(words, I32), new(words, I32)

    def run(self, stream):
        lib, (rows, cols, width), t = self.device.lib, self.shape, self.dtype
        p = lambda b: b.data_ptr()
        o = {n: p(b) for n, b in self.out.items()}
        st = [p(b) for b in self.stats]
        lib.mg_residual_norm_fwd(p(self.f), p(self.h), p(self.gate), p(self.pg), p(self.pb), p(self.ng), p(self.nb), o["h_out"], o["x"], *st,
                                 p(self.f8), p(self.x8), rows, cols, rows, 0.9, 1e-5, t, stream)
        lib.mg_residual_norm_bwd(p(self.dx), p(self.dh_out), None, p(self.f8), o["h_out"], p(self.gate), p(self.pg), p(self.pb), p(self.ng), *st,
                                 o["df"], o["dh"], o["dgate"], o["dpg"], o["dpb"], o["dng"], o["dnb"], rows, cols, rows, 0.9, t, F32, stream)
        lib.mg_linear_bwd_act8(p(self.dy), p(self.x8), p(self.w), o["dx"], o["dw"], o["db"], rows, width, cols, 0, 0, t, F32, stream)

    def clear(self):
        for b in self.out.values():
            self.device.lib.mg_fill(b.data_ptr(), 5.0, b.numel, b.dtype, self.device.stream)

    def read(self):
        return {n: b.to_numpy() for n, b in self.out.items()}


@pytest.mark.parametrize("dtype,route", [(BF16, "0"), (BF16, "1"), (F32, "1")])
def test_graphs_keep_their_scratch(device, monkeypatch, dtype, route):
    monkeypatch.setenv("MOGRAD_HIP_ACT8_ROUTE", route)
    hip = C.CDLL("libamdhip64.so")

    def ok(rc, what):
        assert rc == 0, f"{what}: {rc}"

    rows, cols, width = 700, 96, 72
    works = [_Work(device, 300 + i, rows, cols, width, dtype) for i in range(2)]
    other = _Work(device, 310, rows, cols, width, dtype)
    want = []
    for w in works:
        w.run(device.stream)
        want.append(w.read())
    graphs = []
    for w in works:  # captured in the mode that forbids allocations elsewhere in the process
        before, after = PoolStats(), PoolStats()
        device.lib.mg_pool_get_stats(before)
        graph, run = C.c_void_p(), C.c_void_p()
        ok(hip.hipStreamBeginCapture(device.stream, C.c_int(0)), "hipStreamBeginCapture")
        try:
            w.run(device.stream)
        finally:
            ok(hip.hipStreamEndCapture(device.stream, C.byref(graph)), "hipStreamEndCapture")
        device.lib.mg_pool_get_stats(after)
        assert after.allocated_bytes > before.allocated_bytes, "what the recorded calls took stays taken"
        ok(hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)), "hipGraphInstantiate")
        graphs.append((graph, run))
    for turn in range(3):
        for w in works:
            w.clear()
        filled = [AnyBuffer.create(F32, device, n, fill=float("nan")) for n in (cols, rows, 8 * cols, rows * cols, 40 * cols, 128 * 128, 16 * 128 * 128)]
        for i, (_, run) in enumerate(graphs):
            other.run(device.stream)
            ok(hip.hipGraphLaunch(run, device.stream), "hipGraphLaunch")
            if turn == 1:
                device.synchronize()
            other.run(device.stream)
        for w, values in zip(works, want):
            for n, v in w.read().items():
                assert np.array_equal(v, values[n]), (turn, n)
        del filled
    for graph, run in graphs:
        ok(hip.hipGraphExecDestroy(run), "hipGraphExecDestroy")
        ok(hip.hipGraphDestroy(graph), "hipGraphDestroy")


def test_an_eager_call_gives_its_scratch_back(device):
    w = _Work(device, 320, 300, 64, 40, BF16)
    w.run(device.stream)
    before, after = PoolStats(), PoolStats()
    device.lib.mg_pool_get_stats(before)
    w.run(device.stream)
    device.lib.mg_pool_get_stats(after)
    assert after.allocated_bytes == before.allocated_bytes


def test_another_stream(device):
    """A second stream of the device, ordered behind the first by the host: the calls run where they are told to."""
    stream = C.c_void_p()
    device.lib.mg_stream_create(C.byref(stream))
    w = _Work(device, 330, 300, 200, 40, BF16)
    w.run(device.stream)
    want = w.read()
    w.clear()
    device.synchronize()
    w.run(stream)
    device.lib.mg_stream_sync(stream)
    for n, v in w.read().items():
        assert np.array_equal(v, want[n]), n
    device.lib.mg_stream_destroy(stream)
