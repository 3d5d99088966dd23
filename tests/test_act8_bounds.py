"""What fp32 Linear gradients from 8 bits leave out of the least dY."""
import numpy as np
import pytest

import test_act8 as A
from oracle import oracle_np as O

from mograd_amd import F32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("xe", [-20, 0, 40, 100])
@pytest.mark.parametrize("M,N,K", [(64, 80, 32), (130, 67, 33)])
def test_least_gradients(device, monkeypatch, M, N, K, xe):
    """dY of 2^-70 to 2^-149, one to a column of dw, beside full ones: three bf16 terms hold a value to 2^-133, exactly from 2^-110 on
    (24 bits of a value of 2^-110 and up end at 2^-133).  dw is one product each, so off by that much times |X'|, and half a step, which
    in fp32 is never less than 2^-150."""
    monkeypatch.setenv("MOGRAD_HIP_ACT8_ROUTE", "1")
    x = np.zeros((M, K), np.float32)
    x[5, ::3] = np.float32(1.25 * 2.0 ** xe)
    act8 = O.act8_store(x, "f32")
    assert np.array_equal(O.act8_load(act8, M, K), x)
    dy = A.normal(61, 0, (M, N)).astype(np.float32)  # (of the other rows, whose X' is zero)
    e = np.arange(N) + 149 - (N - 1)
    dy[5] = np.ldexp(1 + np.abs(A.normal(61, 1, N)) % 1, -e).astype(np.float32)
    _, dw, db = A._linear(device, dy, act8, np.zeros((N, K)), M, N, K, F32, F32)
    want = dy[5].astype(np.float64)[:, None] * x[5].astype(np.float64)[None]
    half = np.maximum(2.0 ** -24 * np.abs(want), 2.0 ** -150)
    # three products, added in fp32: each addition may lose half a step of the sum
    bound = 3 * half + np.where(np.abs(dy[5]) < 2.0 ** -110, 2.0 ** -133, 0.0)[:, None] * np.abs(x[5])
    assert (np.abs(dw - want) <= bound).all()
    A._check(db, dy.astype(np.float64).sum(0), A._bound(dy.astype(np.float64).sum(0), np.abs(dy).astype(np.float64).sum(0), M, F32), "db")
