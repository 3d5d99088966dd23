"""What the library asks of the HIP runtime, without a GPU: its host code runs over tests/host_cpp/stub_hip.cpp, in a process of its
own, which writes launches down and refuses those of 2^32 threads along an axis, as the runtime does."""
import json
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

PRELUDE = """
import ctypes as C, json, sys
sys.path.insert(0, sys.argv[2])
stub = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)  # before the library, whose calls it takes
stub.stub_launches.restype = stub.stub_mallocs.restype = C.c_int64
stub.stub_launches.argtypes = [C.c_char_p, C.c_int64]
stub.stub_capture.argtypes = [C.c_ulonglong]
import mograd_amd
from mograd_amd import BF16, F16, F32, MogradError
lib = mograd_amd.load()
p, p16 = C.c_void_p(1 << 20), C.c_void_p((1 << 20) + 2)

def launches():
    n = stub.stub_launches(None, 0)
    text = C.create_string_buffer(n + 1)
    stub.stub_launches(text, n + 1)
    stub.stub_reset()
    return [list(map(int, line.split())) for line in text.value.decode().splitlines()]

def norm_fwd(rows, cols, gate_rows=1, dtype=BF16, post=True, pre=True, keep=None, stream=None):
    o, n = (p if post else None), (p if pre else None)
    lib.mg_residual_norm_fwd(p, p, p, o, o, n, n, p, n, o, o, n, n, keep, keep, rows, cols, gate_rows, 1.0, 1e-5, dtype, stream)

def norm_bwd(rows, cols, gate_rows=1, dtype=BF16, post=True, pre=True, f8=False, stream=None):
    o, n = (p if post else None), (p if pre else None)
    lib.mg_residual_norm_bwd(n, p, None if f8 else p, p if f8 else None, p, p, o, o, n, o, o, n, n, p, p, p, o, o, n, n, rows, cols,
                             gate_rows, 1.0, dtype, F32, stream)

def linear(M, N, K, dtype=BF16, dx=True, relu=1, stream=None):
    lib.mg_linear_bwd_act8(p, p, p, p if dx else None, p, p, M, N, K, 0, relu, dtype, F32, stream)

out = []
"""


@pytest.fixture(scope="module")
def stub_hip(tmp_path_factory):
    out = tmp_path_factory.mktemp("stub") / "libstub_hip.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    str(ROOT / "tests" / "host_cpp" / "stub_hip.cpp"), "-o", str(out)], check=True)
    return out


@pytest.fixture
def over_stub(stub_hip):
    def run(code):
        """`code` over the stub; what it puts into `out`."""
        child = subprocess.run([sys.executable, "-c", PRELUDE + code + "\nprint(json.dumps(out))", str(stub_hip), str(ROOT)],
                               capture_output=True, text=True, timeout=300)
        assert child.returncode == 0, child.stderr[-2000:]
        return json.loads(child.stdout.splitlines()[-1])

    return run


def test_the_stub_takes_the_calls(over_stub):
    got = over_stub("norm_fwd(128, 64); out = launches()")
    assert len(got) == 1 and got[0][3:6] == [256, 1, 1]


def test_residual_norm_of_many_narrow_or_wide_rows(over_stub):
    """Fewer columns than a chunk, or more than registers hold, where a workgroup has a row at a time: any number of rows."""
    got = over_stub("""
for rows in (3, 1 << 22, (1 << 31) - 1):
    for cols, dtype in ((7, BF16), (1, F32), (3, F16), (20001, BF16)):
        for keep in (None, p):
            if rows * cols < 1 << 34:
                norm_fwd(rows, cols, rows, dtype, keep=keep if rows < 1 << 23 else None)
                norm_bwd(rows, cols, rows, dtype)
                out.append(len(launches()))
""")
    assert got and min(got) >= 3


def test_residual_norm_backward_of_the_widest_rows(over_stub):
    """The second stage has 1024 threads for 32 columns; every column of 2^30 - 1 is covered."""
    got = over_stub("""
for cols in (20001, (1 << 27) - 1, 1 << 27, (1 << 30) - 1):
    for post, pre in ((True, True), (False, True)):
        norm_bwd(2, cols, 1, BF16, post, pre)
        stage2 = [l for l in launches() if l[3] == 1024][1:]  # (the first has the rows)
        out.append((cols, sum(l[0] for l in stage2)))
""")
    for cols, groups in got:
        assert groups == -(-cols // 32), cols


def test_act8_of_more_chunks_than_a_launch_counts(over_stub):
    """(2^31 - 1, 1): 2^31 - 1 blocks of 32, four threads' worth or eight each. Every chunk of 16 bytes has its thread."""
    got = over_stub("""
for rows, cols in ((5, 40), ((1 << 29) - 1, 1), ((1 << 31) - 1, 1), ((1 << 31) - 1, 512), (1 << 20, 1 << 20)):
    for dtype in (F32, BF16):
        chunks = rows * -(-cols // 32) * (8 if dtype == F32 else 4)
        each = 4 if chunks >= 1 << 20 else 1
        for call in (lib.mg_act8_store, lib.mg_act8_load):
            call(p, p, rows, cols, *([0] if call is lib.mg_act8_store else []), dtype, None)
            out.append((rows, cols, chunks, each * sum(l[0] * l[3] for l in launches())))
""")
    for rows, cols, chunks, places in got:
        assert 0 <= places - chunks < 4 * 256, (rows, cols)


def test_act8_linear_of_more_tiles_than_a_launch_counts(over_stub):
    """fp32 dX in tiles of 64 rows beside dW: 2^24 of them are 2^32 threads."""
    got = over_stub("""
for M in (1 << 20, (1 << 30) - 64, 1 << 30, 0x7f000000):
    for N, K in ((32, 4), (32, 32), (64, 64)):
        linear(M, N, K, F32)
        out.append(len(launches()))
""")
    assert got and min(got) >= 1


def test_a_recorded_call_that_cannot_keep_its_scratch_is_refused(over_stub):
    """Scratch is kept for the graph under a capture mode of the call's own; without it nothing is taken and nothing launched."""
    got = over_stub("""
stream = C.c_void_p(1 << 16)
stub.stub_capture(7)
norm_bwd(64, 64, 64, stream=stream)
linear(64, 64, 64, stream=stream)
launches()
took = stub.stub_mallocs()
stub.stub_exchange_fails(1)
for call in (lambda: norm_bwd(512, 640, 512, stream=stream), lambda: linear(1024, 640, 512, stream=stream)):
    try:
        call()
        out.append(0)
    except MogradError as e:
        out.append(e.status)
out += [len(launches()), stub.stub_mallocs() - took]
norm_bwd(64, 64, 64)  # (the default stream is never captured)
out.append(len(launches()))
""")
    assert got[:4] == [3, 3, 0, 0] and got[4] > 0


def test_recorded_calls_share_scratch_within_a_stream_of_a_capture(over_stub):
    """A replay runs them in order, so the second takes what the first had; another stream, another capture and eager calls do not, until
    the program has destroyed its graphs and says so."""
    got = over_stub("""
from mograd_amd._lib import PoolStats
streams = C.c_void_p(1 << 16), C.c_void_p(1 << 17)

def both(stream):
    norm_bwd(512, 640, 512, stream=stream)
    linear(1024, 640, 512, stream=stream)

def taken():
    stats = PoolStats()
    lib.mg_pool_get_stats(stats)
    return stats.allocated_bytes

def during(capture, stream):
    stub.stub_capture(capture)
    before = taken()
    both(stream)
    out.append(taken() - before)

during(0, streams[0])
for capture, stream in ((7, 0), (7, 0), (7, 1), (7, 0), (8, 0), (8, 0), (0, 0)):
    during(capture, streams[stream])
out.append(taken())
stub.stub_capture(0)
lib.mg_pool_free_recorded()
out.append(taken())
mallocs = stub.stub_mallocs()
both(streams[0])
out += [taken(), stub.stub_mallocs() - mallocs, stub.stub_mode()]
""")
    eager, first, again, other_stream, back, other_capture, again2, between, held, *rest = got
    assert eager == again == back == again2 == between == 0
    assert first == other_stream == other_capture > 0 and held == 3 * first
    assert rest == [0, 0, 0, 0]


def test_recorded_calls_on_the_streams_of_two_threads(over_stub):
    """hipStreamPerThread is a stream of each thread by one name: as branches of one capture they do not share scratch."""
    got = over_stub("""
import threading
from mograd_amd._lib import PoolStats

def record():
    before, after = PoolStats(), PoolStats()
    lib.mg_pool_get_stats(before)
    linear(1024, 640, 512, stream=C.c_void_p(2))
    lib.mg_pool_get_stats(after)
    out.append(after.allocated_bytes - before.allocated_bytes)

stub.stub_capture(7)
record()
record()
other = threading.Thread(target=record)
other.start()
other.join()
""")
    assert got[0] > 0 and got == [got[0], 0, got[0]]


def test_a_transformer_without_blocks_takes_the_options(over_stub):
    """Embedding and head alone: there is nothing that the options change."""
    got = over_stub("""
import numpy as np
from mograd_amd import AnyBuffer, Device
from mograd_amd.tiny_transformer import TinyTransformer
device = Device()
ids = AnyBuffer.from_numpy(device, np.zeros((2, 8), np.int32))
for options in (dict(), dict(post_norm=True), dict(act8=True), dict(residual_scale=0.5)):
    model = TinyTransformer(device, 17, 32, 64, 0, 2, **options)
    launches()
    model.step(ids, ids, 2, 8)
    out.append((launches(), model.kept_bytes()))
for l in out:
    l[0][:] = [v[:6] for v in l[0]]
""")
    assert len(got[0][0]) > 0 and all(g == got[0] for g in got)


def test_the_header_names_the_entries_that_take_scratch(over_stub):
    """Calls of these that overlap in time on two streams write into each other's scratch; the header's conventions say which."""
    got = over_stub("""
from mograd_amd._lib import PoolStats

def asked():
    stats = PoolStats()
    lib.mg_pool_get_stats(stats)
    return stats.hit_count + stats.miss_count

for name, call in (("mg_act8_store", lambda: lib.mg_act8_store(p, p, 64, 64, 0, BF16, None)),
                   ("mg_act8_load", lambda: lib.mg_act8_load(p, p, 64, 64, BF16, None)),
                   ("mg_linear_bwd_act8", lambda: linear(64, 64, 64)), ("mg_residual_norm_fwd", lambda: norm_fwd(64, 3, 64, keep=p)),
                   ("mg_residual_norm_bwd", lambda: norm_bwd(64, 64, 64))):
    before = asked()
    call()
    out.append((name, asked() > before))
""")
    text = (ROOT / "include" / "mograd_hip.h").read_text()
    conventions = text[text.index("every entry point that takes scratch"):text.index("returns its blocks")]
    for name, takes in got:
        assert (name in conventions) == takes, name
