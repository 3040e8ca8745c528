"""silu(gate) * up over fp32's whole range: large ups with gates so negative that neither gate * up nor exp(-gate) fits fp32, though the value does.

A product here is one term, so gates and ups are exact: the value's error is its arithmetic's, (12 + 1.3 |gate|) 2^-24 (two exp2 and a reciprocal within an ulp, five
products, and exp2's argument, rounded to 1.22 2^-24 of |gate|), and the output's rounding.
"""
import numpy as np
import pytest

from bybylang_amd import _abi, synth
from mx_ref import MX4, MX8, close_mx, codes_of, km, plan, rows
from paged_ref import close, from_bits

pytestmark = pytest.mark.gpu
F32, F16, BF16 = _abi.F32, _abi.F16, _abi.BF16
NP = {F32: np.float32, F16: np.float16, BF16: np.uint16}
GATES = [-52.0, -96.0, -0.25, 2.0, -3.0, -12.0, -26.0, -88.0, 40.0, -60.0, 0.0, -104.0, -120.0, 15.0, -160.0, 1.0]  # 4 significant bits at most


def silu(g):
    return g * np.exp(-np.maximum(-g, 0)) / (1 + np.exp(-np.abs(g)))


def mx(values, exps, fmt):
    """A buffer of rows that hold values [R, K] exactly under the scales 2^exps [R, K / 32]."""
    R, K = values.shape
    codes = km(codes_of(values / 2.0 ** np.repeat(exps, 32, axis=1), fmt))
    if fmt == MX4:
        codes = codes[:, 0::2] | codes[:, 1::2] << 4
    return np.concatenate([codes.reshape(-1), (exps + 127).astype(np.uint8).reshape(-1)])


def operands(M, N, K, up_exp, seed):
    """Rows whose first value is a gate's and whose value 32 is an up's size; matrices that take the one into gates and the other into ups.
    Gates are GATES by row (1 by the matrix), ups +-1.5 2^up_exp by output."""
    g = synth.rng(seed)
    x, xe = np.zeros((M, K)), np.zeros((M, K // 32), int)
    gate = np.array([GATES[i % len(GATES)] for i in range(M)])
    lead = np.floor(np.log2(np.abs(np.where(gate == 0, 1, gate)))).astype(int)
    x[:, 0], xe[:, 0] = gate, lead - 3
    half = up_exp // 2
    x[:, 32], xe[:, 1] = 2.0**half, half
    w, we = np.zeros((2 * N, K)), np.zeros((2 * N, K // 32), int)
    sign = g.choice([-1.0, 1.0], N)
    w[:N, 0] = 1.0
    w[N:, 32], we[N:, 1] = sign * 1.5 * 2.0 ** (up_exp - half), up_exp - half
    up = sign * 1.5 * 2.0**up_exp
    return mx(x, xe, MX8), mx(w, we, MX4), gate, up


def agree(raw, gate, up, yt, M, N):
    want = silu(gate)[:, None] * up
    slack = (12 + 1.3 * np.abs(gate))[:, None] * 2.0**-24 * np.abs(want)
    if yt in (MX8, MX4):
        assert np.all(raw[M * N * (8 if yt == MX8 else 4) // 8:] != 255), "groups marked as not finite"
        close_mx(raw, want, slack, yt)
        return
    got = from_bits(raw.view(NP[yt]).reshape(M, N), yt)
    close(got, want, yt, slack)


# Few rows (moe_rows), and blocks enough for moe_tiles.
@pytest.mark.parametrize("M,N", [(1, 32), (16, 96), (48, 64), (700, 1056)])
@pytest.mark.parametrize("yt,up_exp", [(F32, 122), (F32, -100), (BF16, 122), (MX8, 122), (MX4, 122), (MX8, 0), (F16, 3)])
def test_one_matrix(hip, M, N, yt, up_exp):
    K = 128
    xb, wb, gate, up = operands(M, N, K, up_exp, M)
    assert np.array_equal(rows(xb, M, K, MX8)[:, 0], gate)
    dev = hip.DeviceBuffer.from_array
    y = hip.DeviceBuffer(M * N * 33 // 32 if yt == MX8 else M * N * 17 // 32 if yt == MX4 else M * N * np.dtype(NP[yt]).itemsize)
    hip.mx_matmul(dev(xb), MX8, dev(wb), M, K, N, _abi.MOE_SWIGLU, y, N, yt)
    agree(y.read(np.uint8), gate, up, yt, M, N)


@pytest.mark.parametrize("T,N", [(16, 64), (700, 1056)])
@pytest.mark.parametrize("yt", [F32, BF16, MX8])
def test_experts(hip, T, N, yt):
    K, E, k = 128, 2, 1
    xb, wb, gate, up = operands(T, N, K, 122, 3)
    both = np.concatenate([wb[:2 * N * K // 2], wb[:2 * N * K // 2], wb[2 * N * K // 2:], wb[2 * N * K // 2:]])
    dev = hip.DeviceBuffer.from_array
    ids = (np.arange(T) // 3 % 2).astype(np.int32).reshape(T, 1)
    buf = hip.DeviceBuffer(hip.moe_plan_bytes(T, k, E))
    p = hip.MoePlan(buf, T, k, E)
    hip.moe_plan(dev(ids), p)
    y = hip.DeviceBuffer(T * N * 33 // 32 if yt == MX8 else T * N * np.dtype(NP[yt]).itemsize)
    hip.moe_matmul(dev(xb), MX8, dev(both), p, K, N, _abi.MOE_GATHER | _abi.MOE_SWIGLU, y, N, yt)
    order = plan(ids, E)[1]
    agree(y.read(np.uint8), gate[order], up, yt, T, N)
