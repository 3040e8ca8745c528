"""moe_tiles with fp32 outputs (8-bit rows in two parts) and with fewer blocks than fill the card: rows enough for it, every epilogue. Bounds as in test_mx_gpu.py and
test_moe_gpu.py."""
import pytest

from bybylang_amd import _abi, synth
from mx_ref import MX4, MX8
from test_moe_gpu import check_product
from test_mx_gpu import check

pytestmark = pytest.mark.gpu
F32, F16, BF16 = _abi.F32, _abi.F16, _abi.BF16
GATHER, SCATTER, GLU = _abi.MOE_GATHER, _abi.MOE_SCATTER, _abi.MOE_SWIGLU


@pytest.mark.parametrize("xf", [MX8, MX4])
@pytest.mark.parametrize("M,K,N,pad", [(1541, 128, 2049, 0), (1030, 384, 2945, 3), (1200, 512, 2560, 0), (2000, 640, 1601, 7)])
def test_fp32(hip, xf, M, K, N, pad):
    check(hip, M, K, N, xf, F32, pad=pad, seed=M)


@pytest.mark.parametrize("xf", [MX8, MX4])
@pytest.mark.parametrize("M,K,N,pad", [(1541, 128, 1025, 0), (1030, 384, 1504, 4), (1300, 256, 1281, 1)])
def test_fp32_gates_and_ups(hip, xf, M, K, N, pad):
    check(hip, M, K, N, xf, F32, glu=True, pad=pad, seed=M)


@pytest.mark.parametrize("T,k,E,K,N", [(700, 3, 6, 256, 1568), (1900, 2, 5, 128, 800), (500, 8, 60, 128, 1056)])
@pytest.mark.parametrize("flags", [SCATTER, 0, GATHER, GATHER | GLU, GLU | SCATTER])
def test_fp32_experts(hip, T, k, E, K, N, flags):
    check_product(hip, T, k, E, K, N, MX8, F32, flags, seed=T)


@pytest.mark.parametrize("yt", [F16, MX8, MX4])
@pytest.mark.parametrize("flags", [GATHER | GLU, SCATTER])
def test_exact_experts(hip, flags, yt):
    check_product(hip, 700, 3, 6, 256, 1568, MX8, yt, flags | _abi.MOE_EXACT, seed=1)


@pytest.mark.parametrize("flags,yt", [(SCATTER, F32), (GLU | SCATTER, BF16), (GATHER | GLU, MX8)])
def test_assignments_left_out(hip, flags, yt):
    g = synth.rng(3)
    check_product(hip, 1500, 2, 5, 256, 1056, MX8, yt, flags, ids=g.integers(-2, 7, (1500, 2)).astype("int32"), seed=5)


@pytest.mark.parametrize("yt", [F16, MX8])
@pytest.mark.parametrize("M,N", [(95, 15808), (190, 7904), (120, 12512)])
def test_few_blocks(hip, yt, M, N):
    check(hip, M, 128, N, MX8, yt, seed=M)


@pytest.mark.parametrize("M,K,N", [(33, 2048, 19300), (40, 4096, 8002), (200, 4096, 1701), (300, 2176, 2050), (520, 640, 4001)])
@pytest.mark.parametrize("yt,pad", [(F32, 0), (F16, 0), (BF16, 0), (BF16, 3)])
def test_rows_in_4_bits(hip, M, K, N, yt, pad):
    """Enough products for byhip_mxfp4_gemm's kernels, and the same with rows of y apart, which stay here."""
    check(hip, M, K, N, MX4, yt, pad=pad, seed=M)
