"""Activations in 8 bits at the sizes that only large tensors reach."""
import ctypes as C

import numpy as np
import pytest

import test_act8 as A
from mograd_amd import F32, I32, AnyBuffer

pytestmark = pytest.mark.gpu


def test_more_chunks_than_32_bits_count_and_a_launch_holds(device):
    """(2^30 + 5, 1) fp32: 2^33 + 40 chunks with their padding, of which a launch takes 2^33.  Whole numbers of up to 127 come back as
    they were."""
    lib, s = device.lib, device.stream
    rows, part = (1 << 30) + 5, 251 << 18  # (a part holds whole periods of the values)
    at = lambda buf, byte: C.c_void_p(buf.storage.ptr + byte)
    pattern = np.resize(np.arange(-125, 126, dtype=np.float32), part)
    x, back = (AnyBuffer.create(F32, device, rows + 4) for _ in range(2))
    act8 = AnyBuffer.create(I32, device, -(-lib.mg_act8_bytes(rows, 1) // 4))
    one = AnyBuffer.from_numpy(device, pattern, F32)
    lib.mg_fill(back.data_ptr(), 7.0, rows + 4, F32, s)
    for first in range(0, rows, part):
        lib.mg_copy_device(at(x, 4 * first), one.data_ptr(), 4 * min(part, rows - first), s)
    lib.mg_act8_store(x.data_ptr(), act8.data_ptr(), rows, 1, 0, F32, s)
    lib.mg_act8_load(act8.data_ptr(), back.data_ptr(), rows, 1, F32, s)
    got = np.empty(part, np.float32)
    for first in range(0, rows, part):
        n = min(part, rows - first)
        lib.mg_copy_to_host(got.ctypes.data_as(C.c_void_p), at(back, 4 * first), 4 * n, s)
        assert np.array_equal(got[:n], pattern[:n]), first
    lib.mg_copy_to_host(got.ctypes.data_as(C.c_void_p), at(back, 4 * rows), 16, s)
    assert (got[:4] == 7).all()
    # the last rows' bytes of q, the value times a power of two beside 31 zeros, and the first and last rows' exponents
    tail = np.empty((64, 32), np.int8)
    lib.mg_copy_to_host(tail.ctypes.data_as(C.c_void_p), at(act8, 32 * (rows - 64)), tail.nbytes, s)
    e = np.empty((2, 64), np.uint8)
    for i, row in enumerate((0, rows - 64)):
        lib.mg_copy_to_host(e[i].ctypes.data_as(C.c_void_p), at(act8, 32 * rows + row), 64, s)
    value = lambda first: pattern[(first + np.arange(64)) % 251]
    assert (tail[:, 1:] == 0).all()
    assert np.array_equal(np.ldexp(tail[:, 0].astype(np.float64), e[1].astype(int) - 133), value(rows - 64))
    assert np.array_equal(np.where(value(0) == 0, 7, np.frexp(value(0))[1] + 126), e[0])  # 2^E <= |x| < 2^(E + 1): k = E - 6
    del x, back, act8, one
    lib.mg_pool_empty_cache()


@pytest.mark.parametrize("dtype", A.FLOATS)
@pytest.mark.parametrize("rows,cols", [(-1, 1024), (0, 1024), (1, 1024), (37, 1001), (5, 993)])
def test_four_chunks_a_thread(device, dtype, rows, cols):
    """Tensors of a million chunks of 16 bytes on the way there: one row fewer, just as many, and more, the last workgroup not full."""
    rows += (1 << 20) * (4 if dtype == F32 else 8) // 1024
    A.test_store_and_load(device, dtype, rows, cols, keep_sign=rows % 2)
