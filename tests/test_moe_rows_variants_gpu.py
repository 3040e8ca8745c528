"""The forms of moe_rows that decode steps and few rows run on: windows of 512 values (K from 1408 on), whole and partial, strips of 64 outputs whose last is partly empty, gates and
ups, units of 16, 32 and 64 rows, every output type. Bounds as in test_mx_gpu.py, those of fp32 outputs."""
import functools

import numpy as np
import pytest

from bybylang_amd import _abi, synth
from mx_ref import MX4, MX8, plan, random_rows
from test_mx_gpu import agree, expected, mx_size

pytestmark = pytest.mark.gpu
F32, F16, BF16 = _abi.F32, _abi.F16, _abi.BF16
GATHER, SCATTER, GLU = _abi.MOE_GATHER, _abi.MOE_SCATTER, _abi.MOE_SWIGLU
SIZE = {F32: 4, F16: 2, BF16: 2}


@functools.lru_cache(maxsize=2)
def problem(rows, x_rows, K, xf, seed):
    """(matrices' buffer, their values), (rows' buffer, their values)."""
    g = synth.rng(seed)
    return random_rows(g, rows, K, MX4), random_rows(g, x_rows, K, xf)


def out_bytes(A, N, S, yt):
    return mx_size(A, N, yt) if yt in (MX8, MX4) else A * S * SIZE[yt]


@functools.lru_cache(maxsize=2)
def wide(M, K, N, xf):
    (wb, wv), (xb, xv) = problem(N, M, K, xf, M + N)
    return wb, xb, expected(xv, wv, N, K, False, xf, F32)


@pytest.mark.parametrize("yt,cut", [(F32, 0), (BF16, 31), (F16, 1), (MX8, 0), (MX4, 0)])
@pytest.mark.parametrize("xf", [MX8, MX4])
@pytest.mark.parametrize("M,K,N", [(1, 1664, 12832), (16, 256, 12832), (16, 2176, 12832), (30, 1792, 6432), (60, 1568, 6432), (60, 2176, 6432), (256, 1664, 3360), (150, 2080, 4320)])
def test_strips_of_64(hip, xf, M, K, N, yt, cut):
    """N leaves half of the last strip empty; `cut` outputs fewer end it anywhere. The matrix's last scales are the buffer's last bytes."""
    wb, xb, (want, slack) = wide(M, K, N, xf)
    n = N - cut
    up = hip.DeviceBuffer.from_array
    if cut:
        wb = np.concatenate([wb[:n * K // 2], wb[N * K // 2:N * K // 2 + n * K // 32]])
    size = out_bytes(M, n, n, yt)
    y = up(np.full(size + 16, 0xA5, np.uint8))
    hip.mx_matmul(up(xb), xf, up(wb), M, K, n, 0, y, n, yt)
    raw = y.read(np.uint8, size + 16)
    assert np.all(raw[size:] == 0xA5)
    agree(raw[:size], want[:, :n], slack[:, :n], yt, M, n, n)


@pytest.mark.parametrize("yt", [F32, BF16, MX8, MX4])
@pytest.mark.parametrize("xf", [MX8, MX4])
@pytest.mark.parametrize("T,k,E", [(5, 2, 4), (40, 1, 2), (300, 1, 2)])
@pytest.mark.parametrize("K,N", [(1664, 96), (2048, 80), (2112, 96), (2176, 32)])
def test_gates_and_ups(hip, xf, T, k, E, K, N, yt):
    if yt in (MX8, MX4) and N % 32:
        N = 64
    (wb, wv), (xb, xv) = problem(E * 2 * N, T, K, xf, T + K)
    ids = np.argsort(synth.rng(T).standard_normal((T, E)), axis=1)[:, :k].astype(np.int32)
    up = hip.DeviceBuffer.from_array
    buf = hip.DeviceBuffer(hip.moe_plan_bytes(T, k, E))
    p = hip.MoePlan(buf, T, k, E)
    hip.moe_plan(up(ids), p)
    size = out_bytes(T * k, N, N, yt)
    y = up(np.full(size + 16, 0xA5, np.uint8))
    hip.moe_matmul(up(xb), xf, up(wb), p, K, N, GATHER | GLU, y, N, yt)
    raw = y.read(np.uint8, size + 16)
    assert np.all(raw[size:] == 0xA5)
    offsets, order = plan(ids, E)
    want, slack = np.zeros((T * k, N)), np.zeros((T * k, N))
    for e in range(E):
        at = np.arange(offsets[e], offsets[e + 1])
        if at.size:
            want[at], slack[at] = expected(xv[order[at] // k], wv.reshape(E, 2 * N, K)[e], N, K, True, xf, F32)
    agree(raw[:size], want, slack, yt, T * k, N, N)
