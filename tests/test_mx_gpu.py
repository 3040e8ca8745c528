"""Microscaled rows on the MI355X: byhip_mx_quantize and byhip_norm_block into them, bit for bit or within a rounding, and
byhip_mx_matmul against 64 bits.

Bounds. A product of K terms in fp32, in whatever order the matrix instructions add them, is within (K + 8) 2^-24 of the sum of the
terms' magnitudes. With rows in 8 bits the instructions add eight neighbours (in memory order) first, each cut off 13 bits
below the exponent of the largest of them: another 8 * 2^-13 of each eight's largest term, at most its largest |x| times its
largest |w|. With fp32 outputs only terms of x below 8 times their scale are cut off so, against each other. silu is 1.1-Lipschitz and at most |v|: an error of dg in a gate and du in an up moves silu(g) u by at most
1.1 dg (|u| + du) + |g| du; its own arithmetic is within 2^-20 of it (exp's argument is rounded to 2^-24 of |g| < 16, beyond which silu is g or vanishes).
"""
import numpy as np
import pytest

from bybylang_amd import _abi, synth
from mx_ref import MX4, MX8, close_mx, km, quantize, random_rows, row_bytes, rows, silu
from paged_ref import close, from_bits, norm, to_bits

pytestmark = pytest.mark.gpu
F32, F16, BF16 = _abi.F32, _abi.F16, _abi.BF16
NP = {F32: np.float32, F16: np.float16, BF16: np.uint16}
U = 2.0**-24


def mx_size(R, K, fmt):
    return R * (row_bytes(K, fmt) + K // 32)


def quantized(hip, x, xt, fmt, pad=0, offset=0):
    """The device's rows of x [R, K] (already of type xt), in a buffer with a guard behind it."""
    R, K = x.shape
    wide = np.zeros((R, K + pad), x.dtype)
    wide[:, :K] = x
    flat = np.concatenate([np.zeros(offset, x.dtype), wide.reshape(-1)])
    n = mx_size(R, K, fmt)
    y = hip.DeviceBuffer.from_array(np.full(n + 16, 0xA5, np.uint8))
    src = hip.DeviceBuffer.from_array(flat)
    hip.mx_quantize(At(src, offset * x.itemsize), K + pad, xt, R, K, y, fmt)
    got = y.read(np.uint8, n + 16)
    assert np.all(got[n:] == 0xA5)
    return got[:n]


class At:
    def __init__(self, buf, at):
        self.buf, self.ptr = buf, buf.ptr + at


@pytest.mark.parametrize("fmt", [MX8, MX4])
@pytest.mark.parametrize("xt", [F32, F16, BF16])
@pytest.mark.parametrize("R,K,pad,offset", [(1, 32, 0, 0), (3, 96, 0, 0), (5, 2080, 3, 1), (2, 4096, 32, 0), (70, 160, 4, 4)])
def test_quantize_bits(hip, fmt, xt, R, K, pad, offset):
    g = synth.rng(41 + R + K)
    x = to_bits(g.standard_normal((R, K)) * 2.0 ** g.integers(-9, 9, (R, K // 32)).repeat(32, axis=1), xt)
    assert np.array_equal(quantized(hip, x, xt, fmt, pad, offset), quantize(from_bits(x, xt), fmt)[0])


@pytest.mark.parametrize("fmt", [MX8, MX4])
def test_quantize_borders(hip, fmt):
    """Largest values on and next to the borders between scales, ties between values, every exponent, zeros of both signs."""
    tops = []
    for e in list(range(-149, 128, 3)) + [126, 127]:
        for m in (1.0, 1.5, 1.75, np.nextafter(np.float32(1.5), np.float32(2)), np.nextafter(np.float32(1.75), np.float32(2)), np.nextafter(np.float32(2), np.float32(1))):
            with np.errstate(over="ignore"):
                v = np.float32(np.ldexp(np.float64(m), e))
            if np.isfinite(v) and v > 0:
                tops.append(v)
    x = np.zeros((len(tops), 32), np.float32)
    steps = np.concatenate([np.arange(1, 13) / 4, np.arange(1, 13) / 128, [0.0, -0.0, 0.3]])
    for i, v in enumerate(tops):
        x[i, 0] = -v if i % 2 else v
        unit = np.float64(2.0 ** np.floor(np.log2(np.float64(v))))
        x[i, 1:1 + len(steps)] = np.where(np.abs(steps * unit) <= v, steps * unit, 0) * (1 if i % 3 else -1)
    x = np.concatenate([x, np.zeros((1, 32), np.float32), np.full((1, 32), -0.0, np.float32)])
    assert np.array_equal(quantized(hip, x, F32, fmt), quantize(x, fmt)[0])


@pytest.mark.parametrize("fmt", [MX8, MX4])
def test_quantize_not_finite(hip, fmt):
    x = np.ones((4, 96), np.float32)
    x[0, 40], x[1, 95], x[2, 0], x[3, 33] = np.nan, np.inf, -np.inf, -np.nan
    got = quantized(hip, x, F32, fmt)
    s = got[4 * row_bytes(96, fmt):].reshape(4, 3)
    assert np.array_equal(s == 255, [[0, 1, 0], [0, 0, 1], [1, 0, 0], [0, 1, 0]])
    assert np.array_equal(got, quantize(x, fmt)[0])


def test_quantize_no_rows(hip):
    y = hip.DeviceBuffer.from_array(np.full(64, 7, np.uint8))
    hip.mx_quantize(y, 32, F32, 0, 32, y, MX8)
    assert np.all(y.read(np.uint8, 64) == 7)


@pytest.mark.parametrize("fmt", [MX8, MX4])
@pytest.mark.parametrize("N", [32, 64, 96, 1024, 4096, 5120, 8224, 16384, 32768, 32800])
@pytest.mark.parametrize("M,xt,ht", [(3, F32, F32), (2, BF16, F32), (1, F16, F16)])
def test_norm_into_mx(hip, fmt, N, M, xt, ht):
    """The bound of a norm (a relative error of (56 + N / 1024) 2^-24 of its factor) and a rounding to the format. h keeps its own type's."""
    g = synth.rng(77 + N + M)
    up = hip.DeviceBuffer.from_array
    x, r = to_bits(g.standard_normal((M, N)) * np.exp(g.standard_normal(N)), xt), to_bits(g.standard_normal((M, N)), ht)
    w = (1 + 0.2 * g.standard_normal(N)).astype(np.float32)
    n = mx_size(M, N, fmt)
    y, h, bw = up(np.full(n + 16, 0xA5, np.uint8)), up(np.zeros_like(r)), up(w)
    hip.norm_block(up(x), N, xt, M, N, None, None, 0, up(r), N, 1.0, h, N, ht, hip.Norm(_abi.NORM_RMS, 1e-5, bw), y, N, fmt)
    want = from_bits(x, xt) + from_bits(r, ht)
    slack = 2 * U * np.abs(want)
    close(from_bits(h.read(NP[ht], M * N).reshape(M, N), ht), want, ht, slack, "h")
    f = 1 / np.sqrt((want * want).mean(1, keepdims=True) + 1e-5)
    slack = (64 + N / 1024) * U * f * np.abs(w) * np.abs(want)
    got = y.read(np.uint8, n + 16)
    assert np.all(got[n:] == 0xA5)
    close_mx(got[:n], norm(want, _abi.NORM_RMS, 1e-5, w, None), slack, fmt, "y")


@pytest.mark.parametrize("fmt", [MX8, MX4])
def test_norm_into_mx_whole(hip, fmt):
    """post, gate, residual in place and layer norms, unaligned rows; a NaN stays in its row."""
    M, N, W = 5, 352, 353
    g = synth.rng(99)
    up = hip.DeviceBuffer.from_array
    x, r = g.standard_normal((M, W)).astype(np.float32), g.standard_normal((M, W)).astype(np.float32)
    x[3, 7] = np.nan
    w, b, gt = (g.standard_normal(N).astype(np.float32) for _ in range(3))
    bw, bb, y, br = up(w), up(b), hip.DeviceBuffer(mx_size(M, N, fmt)), up(r)
    layer = hip.Norm(_abi.NORM_LAYER, 1e-5, bw, bb)
    hip.norm_block(up(x), W, F32, M, N, layer, up(gt), 0, br, W, 0.5, br, W, F32, layer, y, N, fmt)
    v = norm(x[:, :N].astype(np.float64), _abi.NORM_LAYER, 1e-5, w, b) * gt + 0.5 * r[:, :N]
    want = norm(v, _abi.NORM_LAYER, 1e-5, w, b)
    got, live = y.read(np.uint8), [0, 1, 2, 4]
    s = got[M * row_bytes(N, fmt):].reshape(M, N // 32)
    assert np.all(s[3] == 255)
    keep = np.concatenate([got[:M * row_bytes(N, fmt)].reshape(M, -1)[live].reshape(-1), s[live].reshape(-1)])
    # every value here is below 64 and passes two norms whose factors are near 1: 2^-13 covers 2^-17 of each
    close_mx(keep, want[live], 2.0**-13 * (1 + np.abs(want[live])), fmt, "y")


# ── products ──


def check(hip, M, K, N, xf, yt, glu=False, pad=0, seed=0, x=None, w=None):
    g = synth.rng(600 + seed)
    up = hip.DeviceBuffer.from_array
    R = 2 * N if glu else N
    xb, xv = random_rows(g, M, K, xf) if x is None else x
    wb, wv = random_rows(g, R, K, MX4) if w is None else w
    S = N if yt in (MX8, MX4) else N + pad
    n = mx_size(M, N, yt) if yt in (MX8, MX4) else M * S * (4 if yt == F32 else 2)
    y = up(np.full(n + 16, 0xA5, np.uint8))
    hip.mx_matmul(up(xb), xf, up(wb), M, K, N, _abi.MOE_SWIGLU if glu else 0, y, S, yt)
    raw = y.read(np.uint8, n + 16)
    assert np.all(raw[n:] == 0xA5), "written past the end"
    want, slack = expected(xv, wv, N, K, glu, xf, yt)
    agree(raw[:n], want, slack, yt, M, N, S)


def expected(xv, wv, N, K, glu, xf, yt):
    v, s = xv @ wv.T, (K + 8) * U * (np.abs(xv) @ np.abs(wv).T)
    if xf == MX8:
        x = np.abs(xv)
        if yt == F32:  # a scale is less than its group's largest value / 224: what is 8 / 224 of that or more is 8 scales or more
            x = np.where(x.reshape(len(x), -1, 32) * 224 >= 8 * x.reshape(len(x), -1, 32).max(2, keepdims=True), 0, x.reshape(len(x), -1, 32)).reshape(x.shape)
        most = [km(a).reshape(len(a), K // 8, 8).max(2) for a in (x, np.abs(wv))]
        s = s + 8 * 2.0**-13 * (most[0] @ most[1].T)
    if not glu:
        return v, s
    (gv, uv), (dg, du) = (v[:, :N], v[:, N:]), (s[:, :N], s[:, N:])
    want = silu(gv) * uv
    return want, 1.1 * dg * (np.abs(uv) + du) + np.abs(gv) * du + 2.0**-20 * np.abs(want)


def agree(raw, want, slack, yt, M, N, S):
    if yt in (MX8, MX4):
        close_mx(raw, want, slack, yt, "product")
        return
    got = raw.view(NP[yt]).reshape(M, S)
    if S > N:
        assert np.all(np.ascontiguousarray(got[:, N:]).view(np.uint8) == 0xA5), "written between rows"
    got = from_bits(got[:, :N], yt)
    if yt == F16:  # 65520 and more round to infinity: a half step past the largest fp16 number; within the slack of it, either
        far = np.where(np.abs(want) >= 65520, np.copysign(np.inf, want), want)
        near = np.abs(np.abs(want) - 65520) <= slack
        want = np.where(near & np.isinf(got), np.copysign(np.inf, want), np.where(near & np.isfinite(got), want, far))
    close(got, want, yt, slack, "product")


@pytest.mark.parametrize("xf", [MX8, MX4])
@pytest.mark.parametrize("M", [1, 3, 16, 17, 32, 33, 64, 65, 129, 300])
@pytest.mark.parametrize("K,N", [(32, 1), (512, 100), (1056, 257)])
def test_rows(hip, xf, M, K, N):
    check(hip, M, K, N, xf, F32, seed=M + K)


@pytest.mark.parametrize("xf", [MX8, MX4])
@pytest.mark.parametrize("K", [32, 64, 96, 128, 160, 256, 384, 480, 512, 544, 640, 1024, 1152, 2048, 2080, 4096, 14336])
@pytest.mark.parametrize("M", [5, 140])
def test_lengths(hip, xf, K, M):
    check(hip, M, K, 96, xf, F32, seed=K)


@pytest.mark.parametrize("xf", [MX8, MX4])
@pytest.mark.parametrize("N", [1, 2, 3, 16, 31, 33, 63, 64, 65, 128, 130, 255, 256, 258, 511, 1000])
@pytest.mark.parametrize("M", [7, 200])
@pytest.mark.parametrize("glu", [False, True])
def test_widths(hip, xf, N, M, glu):
    check(hip, M, 256, N, xf, F32, glu=glu, pad=N % 3, seed=N)


@pytest.mark.parametrize("xf", [MX8, MX4])
@pytest.mark.parametrize("yt", [F32, F16, BF16, MX8, MX4])
@pytest.mark.parametrize("M,K,N", [(1, 512, 64), (19, 256, 96), (50, 416, 160), (150, 640, 416), (257, 1024, 512)])
@pytest.mark.parametrize("glu", [False, True])
def test_outputs(hip, xf, yt, M, K, N, glu):
    check(hip, M, K, N, xf, yt, glu=glu, seed=yt)


@pytest.mark.parametrize("xf", [MX8, MX4])
@pytest.mark.parametrize("K", [128, 256, 384, 512, 640, 896, 1152])
@pytest.mark.parametrize("glu", [False, True])
def test_tiles_lengths(hip, xf, K, glu):
    """Enough blocks of 128 rows and 256 matrix rows for moe_tiles, the last of each not full."""
    check(hip, 6 * 128 + 5, K, (1025 if glu else 2049) + K % 3, xf, F16 if glu else F32, glu=glu, pad=1, seed=K)


@pytest.mark.parametrize("xf", [MX8, MX4])
@pytest.mark.parametrize("yt", [F32, F16, BF16, MX8, MX4])
@pytest.mark.parametrize("M,N,pad", [(900, 2080, 0), (1023, 1824, 8), (385, 4128, 5)])
@pytest.mark.parametrize("glu", [False, True])
def test_tiles_outputs(hip, xf, yt, M, N, pad, glu):
    check(hip, M, 256, N if not glu else -(-N // 64) * 32, xf, yt, glu=glu, pad=pad, seed=yt + M)


@pytest.mark.parametrize("M,K,N", [(65, 128, 1), (200, 256, 2), (129, 384, 3)])
def test_narrow_products_of_rows_in_4_bits(hip, M, K, N):
    check(hip, M, K, N, MX4, F32, seed=N)


@pytest.mark.parametrize("M,K,N", [(3, 96, 70), (200, 512, 70), (40, 128, 70), (700, 384, 2100)])
def test_nan_groups_reach_their_outputs_only(hip, M, K, N):
    """A row's NaN group makes the row NaN, a matrix row's the column, and nothing else; the bytes behind a row are not its own."""
    g = synth.rng(5)
    up = hip.DeviceBuffer.from_array
    xb, xv = random_rows(g, M, K, MX8)
    wb, wv = random_rows(g, N, K, MX4)
    xs, ws = xb[M * K:].reshape(M, -1), wb[N * K // 2:].reshape(N, -1)
    xs[1, 0] = ws[69, -1] = ws[4, 0] = 255
    y = hip.DeviceBuffer(M * N * 4)
    hip.mx_matmul(up(xb), MX8, up(wb), M, K, N, 0, y, N, F32)
    got = y.read(np.float32, M * N).reshape(M, N)
    want = np.zeros((M, N), bool)
    want[1], want[:, [4, 69]] = True, True
    assert np.array_equal(np.isnan(got), want)
    v, s = expected(xv, wv, N, K, False, MX8, F32)
    assert np.all(np.abs(got - v)[~want] <= (s + U * np.abs(v))[~want])


def test_far_scales(hip):
    """Scales at both ends of their range: sums neither vanish nor overflow while they fit in fp32."""
    K, M, N = 256, 2, 33
    g = synth.rng(8)
    xb, _ = random_rows(g, M, K, MX8, spread=0)
    wb, _ = random_rows(g, N, K, MX4, spread=0)
    xb[M * K:], wb[N * K // 2:] = 20, 220
    check(hip, M, K, N, MX8, F32, x=(xb, rows(xb, M, K, MX8)), w=(wb, rows(wb, N, K, MX4)))


def test_same_as_mxfp4_gemm(hip):
    """Rows quantised to 4 bits are what byhip_mxfp4_gemm takes."""
    M, K, N = 40, 512, 96
    g = synth.rng(3)
    up = hip.DeviceBuffer.from_array
    x = g.standard_normal((M, K)).astype(np.float32)
    wb, wv = random_rows(g, N, K, MX4)
    xq, y = hip.DeviceBuffer(mx_size(M, K, MX4)), hip.DeviceBuffer(M * N * 4)
    hip.mx_quantize(up(x), K, F32, M, K, xq, MX4)
    hip.mxfp4_gemm(xq, up(wb), y, F32, M, K, N)
    want, slack = expected(quantize(x, MX4)[1], wv, N, K, False, MX4, F32)
    agree(y.read(np.uint8), want, slack, F32, M, N, N)


def test_refusals(hip):
    up = hip.DeviceBuffer.from_array
    z, small = up(np.zeros(8192, np.float32)), up(np.zeros(4, np.float32))

    def quant(x=z, xs=64, xt=F32, M=4, K=64, y=z, f=MX8):
        hip.mx_quantize(x, xs, xt, M, K, y, f)

    def mm(x=z, xf=MX8, w=z, M=4, K=64, N=32, flags=0, y=z, ys=32, yt=F32):
        hip.mx_matmul(x, xf, w, M, K, N, flags, y, ys, yt)

    def nm(N=64, y=z, ys=64, yt=MX8):
        hip.norm_block(z, 64, F32, 4, N, None, None, 0, None, 0, 1.0, None, 0, F32, hip.Norm(0, 1e-5), y, ys, yt)
    quant(), mm(), nm()
    odd = At(z, 4)
    for call, match, kw in [
            (quant, "-1 rows", {"M": -1}), (quant, "multiple of 32", {"K": 40}), (quant, "0 values", {"K": 0}), (quant, "format 0", {"f": F32}), (quant, "dtype 3", {"xt": 3}),
            (quant, "below its width", {"xs": 60}), (quant, "needs .* bytes", {"y": small}), (quant, "needs .* bytes", {"x": small}), (quant, "16-byte aligned", {"y": odd}),
            (mm, "-1 rows", {"M": -1}), (mm, "rows of 0 values", {"K": 0}), (mm, "0 outputs", {"N": 0}), (mm, "multiple of 32", {"K": 48}), (mm, "format 1", {"xf": F16}),
            (mm, "flags 1", {"flags": 1}), (mm, "flags 8", {"flags": 8}), (mm, "needs .* bytes", {"x": small}), (mm, "needs .* bytes", {"w": small}), (mm, "needs .* bytes", {"y": small}),
            (mm, "16-byte aligned", {"x": odd}), (mm, "16-byte aligned", {"w": odd}), (mm, "below its width", {"ys": 31}), (mm, "multiple of 32", {"N": 33, "ys": 33, "yt": MX8}),
            (mm, "no stride", {"ys": 64, "yt": MX8}), (mm, "dtype 9", {"yt": 9}), (mm, "less than 2 GiB", {"M": 2**21, "K": 1024, "x": ANY}), (mm, "a matrix of", {"N": 2**21, "K": 2048, "ys": 2**21}),
            (nm, "multiple of 32", {"N": 40, "ys": 40}), (nm, "no stride", {"ys": 96}), (nm, "needs .* bytes", {"y": small}), (nm, "16-byte aligned", {"y": odd})]:
        with pytest.raises(_abi.HipBackendError, match=match):
            call(**kw)


class ANY:
    """An address that is not the library's: its size is the caller's to know. No refused call reads it."""
    ptr = 0x1000
