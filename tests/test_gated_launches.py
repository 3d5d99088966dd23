"""What the gated layers ask of the HIP runtime, without a GPU (see test_launches.py): their launches at sizes that one launch cannot
count, and what recorded calls take from the pool."""
from test_launches import over_stub, stub_hip  # noqa: F401  (fixtures)

CALLS = """
from mograd_amd._lib import PoolStats

def forward(M, F, K, dtype=BF16, keep=True, x=p, w=p, stream=None):
    lib.mg_gated_linear_fwd(x, w, p, p, p if keep else None, M, F, K, 0, dtype, stream)

def backward(M, F, K, dtype=BF16, grads=F32, dx=True, db=True, pending=None, stream=None):
    args = (p, p, p, p, p if dx else None, p, p if db else None, M, F, K, 0, 0, dtype, grads)
    if pending is None:
        lib.mg_gated_linear_bwd(*args, stream)
    else:
        lib.mg_gated_linear_bwd_deferred(*args, pending, stream)

def taken():
    stats = PoolStats()
    lib.mg_pool_get_stats(stats)
    return stats.allocated_bytes
"""


def test_a_recorded_deferred_backward_keeps_its_scratch(over_stub):
    """The gradients of the projections, the copies of odd rows and the sums that the list holds: a replay writes them all again, so none
    of it goes to anyone else, also once the list is finished."""
    got = over_stub(CALLS + """
streams = C.c_void_p(1 << 16), C.c_void_p(1 << 17)
pending = C.c_void_p()
lib.mg_deferred_create(C.byref(pending))

def step(stream):
    for shape in ((1000, 101, 77, BF16, F32), (1000, 96, 64, F16, F16), (2048, 512, 784, F32, F32)):
        backward(*shape, pending=pending, stream=stream)
    lib.mg_finish_deferred(pending, stream)

def during(capture, stream):
    stub.stub_capture(capture)
    before = taken()
    step(stream)
    out.append(taken() - before)

before = taken()
for capture, stream in ((0, 0), (7, 0), (7, 0), (7, 1), (0, 0), (8, 0), (0, 0)):
    during(capture, streams[stream])
stub.stub_capture(0)
out.append(taken() - before)
mallocs = stub.stub_mallocs()
step(streams[0])  # (eager ones share the pool's)
out.append(stub.stub_mallocs() - mallocs)
lib.mg_pool_free_recorded()
out.append(taken() - before)

# a list that is still pending when the graphs are gone
stub.stub_capture(9)
backward(1000, 101, 77, BF16, F32, pending=pending, stream=streams[0])
stub.stub_capture(0)
lib.mg_pool_free_recorded()
lib.mg_finish_deferred(pending, None)
out.append(taken() - before)
lib.mg_deferred_destroy(pending)
""")
    eager, first, again, other_stream, between, other_capture, after, held, mallocs, freed, rest = got
    assert eager == again == between == after == mallocs == freed == rest == 0
    assert first == other_stream == other_capture > 0 and held == 3 * first


def test_a_recorded_deferred_backward_that_cannot_keep_its_scratch_is_refused(over_stub):
    got = over_stub(CALLS + """
stream, pending = C.c_void_p(1 << 16), C.c_void_p()
lib.mg_deferred_create(C.byref(pending))
stub.stub_capture(7)
stub.stub_exchange_fails(1)
try:
    backward(1000, 101, 77, pending=pending, stream=stream)
    out.append(0)
except MogradError as e:
    out.append(e.status)
out += [len(launches()), stub.stub_mallocs()]
""")
    assert got == [3, 0, 0]


def test_copies_of_more_chunks_than_a_launch_counts(over_stub):
    """Odd rows are copied to rows on chunks, a thread a chunk of 16 bytes: 2^24 workgroups of 256 are 2^32 threads.  Every chunk has its
    thread, also in the other products that make such copies."""
    got = over_stub(CALLS + """
def chunks(rows, cols):
    unit = 64 if cols >= 2048 else 8
    return -(-rows * (-(-cols // unit) * unit // 8) // 256)

for M, F, K in ((1001, 8192, (1 << 22) - 71), (8192, 1001, (1 << 22) - 71), (1001, 1 << 20, 65537), ((1 << 31) - 1, 1, 17)):
    forward(M, F, K)
    out.append((chunks(M, K) + chunks(2 * F, K), sum(l[0] for l in launches()[:-1])))
lib.mg_matmul_bt(p, p, p, 1, 1 << 25, 129, 2051, 2051, 1, 2051, 1, 0, 0, BF16, None)
out.append((chunks(1 << 25, 2051) + chunks(129, 2051), sum(l[0] for l in launches()[:-1])))
""")
    assert len(got) == 5
    for least, given in got:
        assert least >= 1 << 24 and least <= given <= least + 1
