"""Gated layers, rotary positions, the norm of gradients and clipping recorded into HIP graphs, where those that take scratch keep what
they took, and on another stream.

Each graph holds one pass of all of them; it is replayed with eager calls on other inputs, allocations that fill what the pool hands out,
and synchronizations in between, and every replay gives the eager call's bits.
"""
import ctypes as C

import numpy as np
import pytest

from helpers import normal

pytestmark = pytest.mark.gpu

from mograd_amd import BF16, F16, F32, AnyBuffer  # noqa: E402
from mograd_amd._lib import PoolStats  # noqa: E402
from mograd_amd.runtime import round_to_dtype  # noqa: E402


class _Work:
    """One pass on inputs of a seed, with buffers of its own."""

    def __init__(self, device, seed, M, F, K, dtype):
        self.device, self.shape, self.dtype = device, (M, F, K), dtype
        put = lambda i, shape, std=1.0: AnyBuffer.from_numpy(device, round_to_dtype(normal(seed, i, shape, std), dtype), dtype)
        self.x, self.w, self.dy = put(0, (M, K)), put(1, (2 * F, K), K ** -0.5), put(2, (M, F))
        new = lambda n, t=dtype: AnyBuffer.create(t, device, n, fill=0.0)
        self.out = {"y": new(M * F), "gu": new(2 * M * F), "dx": new(M * K), "dw": new(2 * F * K), "dw32": new(2 * F * K, F32), "db": new(2 * F),
                    "db32": new(2 * F, F32), "turned": new(M * (K // 8 * 8)), "norm": new(1, F32), "norm2": new(1, F32), "clipped": new(2 * F * K), "clipped_db": new(2 * F)}
        self.freq = AnyBuffer.from_numpy(device, np.array([1.0, 0.1, 0.01, 0.001], np.float32), F32)

    def run(self, stream):
        lib, (M, F, K), t = self.device.lib, self.shape, self.dtype
        o = {n: b.data_ptr() for n, b in self.out.items()}
        p = lambda b: b.data_ptr()
        lib.mg_gated_linear_fwd(p(self.x), p(self.w), None, o["y"], o["gu"], M, F, K, 0, t, stream)
        lib.mg_gated_linear_bwd(p(self.dy), o["gu"], p(self.x), p(self.w), o["dx"], o["dw"], o["db"], M, F, K, 0, 0, t, t, stream)
        lib.mg_gated_linear_bwd(p(self.dy), o["gu"], p(self.x), p(self.w), None, o["dw32"], o["db32"], M, F, K, 0, 0, t, F32, stream)
        st = (C.c_int64 * 3)(0, K // 8 * 8, 8)
        lib.mg_rotary(p(self.x), o["turned"], None, p(self.freq), None, 1, M, K // 8, 8, 8, st, st, None, 1, 0, 0, 0, t, stream)
        numels, types = (C.c_int64 * 2)(2 * F * K, 2 * F), (C.c_int * 2)(t, t)
        grads, out = ((C.c_void_p * 2)(o[a].value, o[b].value) for a, b in (("dw", "db"), ("clipped", "clipped_db")))
        lib.mg_grad_norm(grads, numels, types, 2, o["norm2"], stream)
        lib.mg_clip_grads(grads, out, numels, types, 2, 0.5, o["norm"], stream)

    def clear(self):
        for b in self.out.values():
            self.device.lib.mg_fill(b.data_ptr(), 5.0, b.numel, b.dtype, self.device.stream)

    def read(self):
        return {n: b.to_numpy() for n, b in self.out.items()}


# the forward's K ranges, ragged copies, the fp32 product that keeps no projections; each takes scratch
CASES = [(BF16, 60, 40, 4096, "64", "4"), (F16, 300, 70, 333, "128", "1"), (F32, 200, 96, 264, "0", "1")]


@pytest.mark.parametrize("dtype,M,F,K,tile,splits", CASES)
def test_graphs_keep_their_scratch(device, monkeypatch, dtype, M, F, K, tile, splits):
    if tile != "0":
        monkeypatch.setenv("MOGRAD_HIP_GATED_TILE", tile)
        monkeypatch.setenv("MOGRAD_HIP_GATED_SPLITS", splits)
    hip = C.CDLL("libamdhip64.so")

    def ok(rc, what):
        assert rc == 0, f"{what}: {rc}"

    works = [_Work(device, 700 + i, M, F, K, dtype) for i in range(2)]
    other = _Work(device, 710, M, F, K, dtype)
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
    sizes = (8, 100, F, M, 2 * M * F, 2 * F * K, 4 * 64 * 64, 64 * 64 * 64, 16 * 128 * 128)
    for turn in range(3):
        for w in works:
            w.clear()
        filled = [AnyBuffer.create(F32, device, n, fill=float("nan")) for n in sizes]
        for _, run in graphs:
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
    device.synchronize()
    device.lib.mg_pool_free_recorded()


def test_an_eager_pass_gives_its_scratch_back(device):
    w = _Work(device, 720, 300, 64, 40, BF16)
    w.run(device.stream)
    before, after = PoolStats(), PoolStats()
    device.lib.mg_pool_get_stats(before)
    w.run(device.stream)
    device.lib.mg_pool_get_stats(after)
    assert after.allocated_bytes == before.allocated_bytes


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_another_stream(device, dtype):
    """A second stream of the device, ordered behind the first by the host: the calls run where they are told to."""
    stream = C.c_void_p()
    device.lib.mg_stream_create(C.byref(stream))
    w = _Work(device, 730, 300, 40, 200, dtype)
    w.run(device.stream)
    want = w.read()
    w.clear()
    device.synchronize()
    w.run(stream)
    device.lib.mg_stream_sync(stream)
    for n, v in w.read().items():
        assert np.array_equal(v, want[n]), n
    device.lib.mg_stream_destroy(stream)
