"""Sizes at which offsets pass 31 and 32 bits: all experts' matrices together, one matrix and one call's rows next to 2 GiB, an output past 2 GiB."""
import numpy as np
import pytest

from bybylang_amd import _abi, synth
from mx_ref import MX4, MX8, plan, random_rows
from paged_ref import close, from_bits
from test_mx_gpu import expected, mx_size

pytestmark = pytest.mark.gpu
F32, BF16 = _abi.F32, _abi.BF16
GATHER, SCATTER, GLU = _abi.MOE_GATHER, _abi.MOE_SCATTER, _abi.MOE_SWIGLU
E, R, K = 17, 131072, 2048
USED = [0, 15, 16]
ROWS = np.array([0, 1, 63, 255, 256, 40000, 65535, 65536, 65537, 105536, 131070, 131071])


@pytest.fixture(scope="module")
def matrices(hip):
    """17 matrices of 128 MiB of values, all zeros but for some rows of the first and the last two."""
    w = hip.DeviceBuffer(mx_size(E * R, K, MX4))
    w.zero()
    values = {}
    for e in USED:
        b, values[e] = random_rows(synth.rng(e), len(ROWS), K, MX4)
        codes, scales = b[:len(ROWS) * K // 2].reshape(len(ROWS), -1), b[len(ROWS) * K // 2:].reshape(len(ROWS), -1)
        for r, c, s in zip(ROWS, codes, scales):
            w.upload(c, (e * R + r) * K // 2)
            w.upload(s, E * R * K // 2 + (e * R + r) * K // 32)
    yield w, values
    w.close()


@pytest.mark.parametrize("xf", [MX8, MX4])
@pytest.mark.parametrize("T,glu,yt", [(5, False, F32), (5, True, BF16), (200, False, BF16), (200, True, F32)])
def test_matrices_past_2_gib(hip, matrices, xf, T, glu, yt):
    """A few rows (moe_rows) and blocks enough for moe_tiles, over matrices that lie past 2^31 bytes."""
    w, values = matrices
    N = R // 2 if glu else R
    xb, xv = random_rows(synth.rng(T), T, K, xf)
    ids = np.array([USED[i % 3] for i in range(T)], np.int32).reshape(T, 1)
    up = hip.DeviceBuffer.from_array
    buf = hip.DeviceBuffer(hip.moe_plan_bytes(T, 1, E))
    p = hip.MoePlan(buf, T, 1, E)
    hip.moe_plan(up(ids), p)
    y = hip.DeviceBuffer(T * N * (4 if yt == F32 else 2))
    hip.moe_matmul(up(xb), xf, w, p, K, N, GATHER | SCATTER | (GLU if glu else 0), y, N, yt)
    got = from_bits(y.read(np.float32 if yt == F32 else np.uint16).reshape(T, N), yt)
    rest = np.ones(N, bool)
    rest[ROWS % N] = False
    assert not got[:, rest].any()
    at = np.unique(ROWS % N)
    for e in USED:
        mine = np.flatnonzero(ids[:, 0] == e)
        full = np.zeros((2 if glu else 1, N, K))
        full.reshape(-1, K)[ROWS] = values[e]
        want, slack = expected(xv[mine], np.concatenate([f[at] for f in full]), len(at), K, glu, xf, yt)
        close(got[np.ix_(mine, at)], want, yt, slack)


def test_an_output_past_2_gib(hip, matrices):
    w, values = matrices
    T = 4300
    xb, xv = random_rows(synth.rng(T), T, K, MX8, spread=0)
    ids = np.array([USED[i % 3] for i in range(T)], np.int32).reshape(T, 1)
    up = hip.DeviceBuffer.from_array
    buf = hip.DeviceBuffer(hip.moe_plan_bytes(T, 1, E))
    p = hip.MoePlan(buf, T, 1, E)
    hip.moe_plan(up(ids), p)
    y = hip.DeviceBuffer(T * R * 4)
    hip.moe_matmul(up(xb), MX8, w, p, K, R, 0, y, R, F32)
    order = plan(ids, E)[1]
    for i in (0, 1432, 1434, 4095, 4096, 4299):
        got = y.read(np.float32, R, i * R * 4)
        e = int(ids[order[i], 0])
        want, slack = expected(xv[i:i + 1], values[e], len(ROWS), K, False, MX8, F32)
        close(got[ROWS][None], want, F32, slack, f"row {i}")
        got[ROWS] = 0
        assert not got.any()


def test_a_matrix_next_to_2_gib_is_taken(hip):
    """The limit is 2^31 bytes of values, not some rows below it: the call goes on to find its matrix too short."""
    z = hip.DeviceBuffer.from_array(np.zeros(4096, np.float32))
    with pytest.raises(_abi.HipBackendError, match="matrices of a product needs 2281700288 bytes"):
        hip.mx_matmul(z, MX8, z, 1, 2048, 2**21 - 1, 0, z, 2**21 - 1, F32)
    with pytest.raises(_abi.HipBackendError, match="a matrix of 2097152 rows"):
        hip.mx_matmul(z, MX8, z, 1, 2048, 2**21, 0, z, 2**21, F32)


def test_rows_of_2_to_the_25_values(hip):
    """More than 64 rows in 4 bits whose offsets do not fit mxfp4_gemm, but are below 2 GiB."""
    M, N, K = 65, 1, 2**25
    kb, kg = K // 2, K // 32
    x, w = hip.DeviceBuffer(M * (kb + kg)), hip.DeviceBuffer(N * (kb + kg))
    x.zero(), w.zero()
    g = synth.rng(1)
    at = [0, 128, K // 2, K - 128]  # stretches of 128 values
    xv, wv = np.zeros((M, 512)), np.zeros((N, 512))
    for i, k in enumerate(at):
        for buf, rows, v in ((x, M, xv), (w, N, wv)):
            b, v[:, 128 * i:128 * i + 128] = random_rows(g, rows, 128, MX4)
            for r in range(rows):
                buf.upload(b[64 * r:64 * r + 64], r * kb + k // 2)
                buf.upload(b[64 * rows + 4 * r:64 * rows + 4 * r + 4], rows * kb + r * kg + k // 32)
    y = hip.DeviceBuffer(M * N * 4)
    hip.mx_matmul(x, MX4, w, M, K, N, 0, y, N, F32)
    # 512 terms that are not 0, in any order among zeros
    close(y.read(np.float32).reshape(M, N), xv @ wv.T, F32, 520 * 2.0**-24 * (np.abs(xv) @ np.abs(wv).T))
