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


def test_sizes_that_a_walk_cannot_count_are_refused(over_stub):
    """Ranges of a walk end on whole steps, past 2^31 where the walk is that long: K of the forward, M and 2 F of the gradients."""
    got = over_stub(CALLS + """
def status(call, *args, **kw):
    try:
        call(*args, **kw)
        return 0
    except MogradError as e:
        return e.status

most = 0x7fff0000
for dtype in (F32, BF16):
    for dx, db in ((True, True), (False, False)):
        for extra, want in ((0, 0), (1, 1)):
            out.append((status(backward, most + extra, 1, 1, dtype, dx=False, db=db), want))
            out.append((status(backward, 1, most // 2 + extra, 1, dtype, dx=dx, db=False), want if extra else None))
    out.append((status(backward, (1 << 31) - 1, 1, 1, dtype, dx=False), 1))
for M, F in ((1, 1), (4, 2), (17, 1)):
    out += [(status(forward, M, F, most, F32), 0), (status(forward, M, F, most + 1, F32), 1), (status(forward, M, F, (1 << 31) - 1, F32), 1)]
out.append((status(forward, (1 << 31) - 1, 1, 17), 0))
""")
    for i, (status, want) in enumerate(got):
        assert want is None or status == want, i


def test_sizes_up_to_2_28_are_taken(over_stub):
    """Every launch counts its threads, whatever is large, as long as the tensors are a card's."""
    got = over_stub(CALLS + """
import random
rng = random.Random(3)
near = lambda: max(1, min(1 << 28, int(2.0 ** rng.uniform(0, 28.2)) + rng.choice((0, 0, 1, -1))))
for _ in range(6000):
    M, F, K, dtype, odd = near(), near(), near(), rng.choice((F32, F16, BF16)), rng.random() < 0.3
    size = 4 if dtype == F32 else 2
    if dtype != F32:
        K = min(K, (1 << 22) - 64)
    if size * (M * K + 2 * F * K + 3 * M * F) > 200e9:
        continue
    q = p16 if odd and dtype != F32 else p
    try:
        forward(M, F, K, dtype, keep=rng.random() < 0.5, x=q, w=q)
        if size * (2 * M * K + 2 * F * K + 5 * M * F) < 200e9:
            backward(M, F, K, dtype, rng.choice((dtype, F32)), dx=rng.random() < 0.7, db=rng.random() < 0.7)
        launches()
        out.append(0)
    except MogradError as e:
        out.append((M, F, K, dtype, odd, str(e)))
""")
    assert len(got) > 2000 and not any(got), [g for g in got if g][:5]
