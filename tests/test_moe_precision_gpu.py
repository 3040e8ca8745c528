"""Products of 8-bit rows enter sums with fp32's precision whatever the output's type, with few rows per matrix (moe_rows) always, with many (moe_tiles) where the caller asks
for it, so that sums whose large terms cancel keep the small ones.

Each eight neighbours of a row here (in memory order, which the instructions add first) hold 448, -448 under equal matrix values and six values below 1/2. The pair's
products cancel exactly, so the bound is that of fp32 outputs (test_mx_gpu.py) for the six alone; a cut 13 bits below the pair's products would leave next to
nothing of them.
"""
import numpy as np
import pytest

from bybylang_amd import _abi, synth
from mx_ref import MX4, MX8, plan, quantize, random_rows
from test_mx_gpu import agree, expected, mx_size

pytestmark = pytest.mark.gpu
F32, F16, BF16 = _abi.F32, _abi.F16, _abi.BF16
GATHER, SCATTER, GLU, EXACT = _abi.MOE_GATHER, _abi.MOE_SCATTER, _abi.MOE_SWIGLU, _abi.MOE_EXACT


def cancelling(g, M, R, K):
    """(rows' buffer, the rows without the pairs), (matrices' buffer, the matrices)."""
    x = g.integers(-8, 9, (M, K // 32, 32)) * 2.0**-5
    w = g.choice([-1.0, -0.5, 0.5, 1.0, 2.0], (R, K // 32, 32))
    x[..., 0:16:4], x[..., 16:32:4] = 448.0, -448.0  # elements e and e + 16 are neighbours in memory
    w[..., 0:16:4] = w[..., 16:32:4] = 6.0
    xb, xv = quantize(x.reshape(M, K), MX8)
    assert np.array_equal(xv, x.reshape(M, K))
    return (xb, np.where(np.abs(xv) == 448, 0, xv)), quantize(w.reshape(R, K), MX4)


@pytest.mark.parametrize("M,K,N", [(1, 256, 32), (7, 2048, 64), (16, 512, 14336), (30, 1024, 96), (60, 96, 64)])
@pytest.mark.parametrize("yt", [F32, F16, BF16, MX8, MX4])
@pytest.mark.parametrize("glu", [False, True])
def test_one_matrix(hip, M, K, N, yt, glu):
    g = synth.rng(M + K)
    (xb, xv), (wb, wv) = cancelling(g, M, 2 * N if glu else N, K)
    n = mx_size(M, N, yt) if yt in (MX8, MX4) else M * N * (4 if yt == F32 else 2)
    y = hip.DeviceBuffer(n)
    hip.mx_matmul(hip.DeviceBuffer.from_array(xb), MX8, hip.DeviceBuffer.from_array(wb), M, K, N, GLU if glu else 0, y, N, yt)
    want, slack = expected(xv, wv, N, K, glu, MX8, F32)
    agree(y.read(np.uint8, n), want, slack, yt, M, N, N)


@pytest.mark.parametrize("yt", [F16, BF16, MX8, MX4])
@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("M,K,N", [(1541, 256, 2112)])
def test_tiles(hip, M, K, N, yt, glu):
    N = N // 2 if glu else N
    g = synth.rng(K)
    (xb, xv), (wb, wv) = cancelling(g, M, 2 * N if glu else N, K)
    n = mx_size(M, N, yt) if yt in (MX8, MX4) else M * N * 2
    y = hip.DeviceBuffer(n)
    hip.mx_matmul(hip.DeviceBuffer.from_array(xb), MX8, hip.DeviceBuffer.from_array(wb), M, K, N, (GLU if glu else 0) | EXACT, y, N, yt)
    want, slack = expected(xv, wv, N, K, glu, MX8, F32)
    agree(y.read(np.uint8, n), want, slack, yt, M, N, N)


def test_flags(hip):
    """4-bit rows are exact as they are and take the flag too; the next bit is refused."""
    g = synth.rng(2)
    (xb, xv), (wb, wv) = random_rows(g, 3, 64, MX4), random_rows(g, 32, 64, MX4)
    x, w, y = hip.DeviceBuffer.from_array(xb), hip.DeviceBuffer.from_array(wb), hip.DeviceBuffer(3 * 32 * 4)
    hip.mx_matmul(x, MX4, w, 3, 64, 32, EXACT, y, 32, F32)
    agree(y.read(np.uint8), *expected(xv, wv, 32, 64, False, MX4, F32), F32, 3, 32, 32)
    with pytest.raises(_abi.HipBackendError, match="flags 32"):
        hip.mx_matmul(x, MX4, w, 3, 64, 32, 32, y, 32, F32)


@pytest.mark.parametrize("T,k,E,K,N", [(3, 2, 8, 2048, 64), (40, 4, 16, 512, 96), (900, 2, 3, 128, 1696)])
@pytest.mark.parametrize("flags,yt", [(GATHER | GLU | EXACT, MX8), (SCATTER | EXACT, BF16), (EXACT, F16), (GATHER | GLU | EXACT, MX4)])
def test_experts(hip, T, k, E, K, N, flags, yt):
    g = synth.rng(T)
    R = 2 * N if flags & GLU else N
    rows = T if flags & GATHER else T * k
    (xb, xv), (wb, wv) = cancelling(g, rows, E * R, K)
    ids = np.argsort(g.standard_normal((T, E)), axis=1)[:, :k].astype(np.int32)
    up = hip.DeviceBuffer.from_array
    buf = hip.DeviceBuffer(hip.moe_plan_bytes(T, k, E))
    p = hip.MoePlan(buf, T, k, E)
    hip.moe_plan(up(ids), p)
    n = mx_size(T * k, N, yt) if yt in (MX8, MX4) else T * k * N * 2
    y = hip.DeviceBuffer(n)
    hip.moe_matmul(up(xb), MX8, up(wb), p, K, N, flags, y, N, yt)
    offsets, order = plan(ids, E)
    want, slack = np.zeros((T * k, N)), np.zeros((T * k, N))
    for e in range(E):
        at = np.arange(offsets[e], offsets[e + 1])
        if at.size:
            a = order[at]
            out = a if flags & SCATTER else at
            want[out], slack[out] = expected(xv[a // k if flags & GATHER else at], wv.reshape(E, R, K)[e], N, K, bool(flags & GLU), MX8, F32)
    agree(y.read(np.uint8, n), want, slack, yt, T * k, N, N)
