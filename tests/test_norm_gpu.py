"""byhip_norm_block against the norms in 64 bits, through device.norm_block.

Bounds: a norm's factor f = 1 / sqrt(mean square + eps) comes from a sum of fp32 terms, at most 32 in a row per
thread (the long form: N / 1024) and 16 more levels, so its relative error is under (48 + N / 1024) / 2 units of
2^-24; the mean's error is that much of the row's mean magnitude. With a few roundings of the value itself: u f |w|
(|v| + mean |v|) for u = (56 + N / 1024) 2^-24. What post gets wrong, pre scales by its own f |w|.
"""
import numpy as np
import pytest

from bybylang_amd import _abi, synth
from paged_ref import close, from_bits, norm, to_bits

pytestmark = pytest.mark.gpu
F32, F16, BF16 = _abi.F32, _abi.F16, _abi.BF16
RMS, LAYER = _abi.NORM_RMS, _abi.NORM_LAYER
NP = {F32: np.float32, F16: np.float16, BF16: np.uint16}
EPS = 1e-5


def factor(v, kind):
    d = v - (v.mean(1, keepdims=True) if kind == LAYER else 0)
    return 1 / np.sqrt((d * d).mean(1, keepdims=True) + EPS)


def run(hip, M, N, xt, ht, yt, post, pre, gate, res, seed=0, pad=0, scale=0.7, in_place=False, affine=True, want_h=True, offset=0.0):
    g = synth.rng(5200 + seed)
    W = N + pad
    up = hip.DeviceBuffer.from_array
    x = to_bits(g.standard_normal((M, W)) + offset, xt)
    r = to_bits(2 * g.standard_normal((M, W)), ht)
    w = [(1 + 0.2 * g.standard_normal(N)).astype(np.float32) for _ in range(2)]
    b = [(0.1 * g.standard_normal(N)).astype(np.float32) for _ in range(2)]
    gt = (0.5 * g.standard_normal((M if gate == "rows" else 1, W))).astype(np.float32)
    keep = [up(a) for a in w + b] + [up(gt)]
    norms = [None if k is None else hip.Norm(k, EPS, keep[i] if affine else None, keep[2 + i] if affine and k == LAYER else None) for i, k in enumerate((post, pre))]
    bx, br = up(x), up(r)
    bh = br if in_place else up(np.zeros_like(r))
    by = hip.DeviceBuffer(M * W * (4 if yt == F32 else 2))
    hip.norm_block(bx, W, xt, M, N, norms[0], keep[4] if gate else None, W if gate == "rows" else 0, br if res else None, W, scale,
                   bh if want_h else None, W, ht, norms[1], by, W, yt)
    u = (56 + N / 1024) * 2.0**-24
    v = from_bits(x, xt)[:, :N]
    slack = np.zeros_like(v)

    def one(v, slack, kind, i):
        wi, bi = (w[i], b[i] if kind == LAYER else None) if affine else (None, None)
        f, aw = factor(v, kind), np.abs(wi) if affine else 1.0
        carried = f * aw * (slack + np.sqrt((slack * slack).mean(1, keepdims=True)) * (1 + f * np.abs(v)))
        return norm(v, kind, EPS, wi, bi), carried + u * f * aw * (np.abs(v) + np.abs(v).mean(1, keepdims=True)) + 2.0**-23 * (0.5 if kind == LAYER else 0)
    if post is not None:
        v, slack = one(v, slack, post, 0)
    if gate:
        gv = gt[:, :N].astype(np.float64)
        slack = slack * np.abs(gv) + 2.0**-23 * np.abs(v * gv)
        v = v * gv
    if res:
        s = float(np.float32(scale)) * from_bits(r, ht)[:, :N]
        slack = slack + 2.0**-23 * (np.abs(s) + np.abs(v))
        v = s + v
    if want_h:
        close(from_bits(bh.read(NP[ht], M * W).reshape(M, W), ht)[:, :N], v, ht, slack, "h")
    if pre is not None:
        y, slack = one(v, slack, pre, 1)
        close(from_bits(by.read(NP[yt], M * W).reshape(M, W), yt)[:, :N], y, yt, slack, "y")


@pytest.mark.parametrize("N", [1, 2, 3, 64, 255, 512, 513, 1000, 4096, 5120, 8191, 8192, 8196, 16384, 32768, 32772, 40001])
@pytest.mark.parametrize("post,pre", [(RMS, RMS), (LAYER, LAYER)])
def test_lengths(hip, N, post, pre):
    run(hip, 3, N, F32, F32, F32, post, pre, "one", True, seed=N)


@pytest.mark.parametrize("xt", [F32, F16, BF16])
@pytest.mark.parametrize("ht", [F32, F16, BF16])
@pytest.mark.parametrize("yt", [F32, F16, BF16])
def test_types(hip, xt, ht, yt):
    run(hip, 5, 768, xt, ht, yt, RMS, LAYER, "rows", True, seed=xt * 9 + ht * 3 + yt)


@pytest.mark.parametrize("kw", [
    dict(post=None, pre=RMS, gate=None, res=True), dict(post=None, pre=LAYER, gate="one", res=False), dict(post=RMS, pre=None, gate="rows", res=True),
    dict(post=None, pre=None, gate="one", res=True), dict(post=RMS, pre=RMS, gate=None, res=True, want_h=False), dict(post=RMS, pre=LAYER, gate=None, res=True, affine=False),
    dict(post=LAYER, pre=RMS, gate="one", res=True, in_place=True)])
@pytest.mark.parametrize("N,pad", [(320, 0), (321, 0), (320, 1), (640, 64), (33000, 0)])
def test_parts_and_strides(hip, kw, N, pad):
    run(hip, 4, N, F16, F32, F16, kw["post"], kw["pre"], kw["gate"], kw["res"], seed=N + pad, pad=pad, **{k: v for k, v in kw.items() if k not in ("post", "pre", "gate", "res")})


def test_many_rows_and_far_means(hip):
    """A mean of 100 deviations: the variance is not lost in it."""
    run(hip, 700, 130, F32, F32, F32, LAYER, LAYER, None, False, seed=1, offset=100.0)
    run(hip, 1, 4096, F32, F32, F32, LAYER, RMS, None, True, seed=2, offset=30.0)


def test_zero_rows_and_constant_rows(hip):
    up = hip.DeviceBuffer.from_array
    y = up(np.full(64, 9, np.float32))
    hip.norm_block(up(np.zeros(64, np.float32)), 64, F32, 0, 64, None, None, 0, None, 0, 0.0, None, 64, F32, hip.Norm(RMS, EPS), y, 64, F32)
    assert np.all(y.read(np.float32) == 9)
    for kind, want in ((LAYER, 0.0), (RMS, 3 / np.sqrt(9 + EPS))):
        hip.norm_block(up(np.full(64, 3, np.float32)), 64, F32, 1, 64, None, None, 0, None, 0, 0.0, None, 64, F32, hip.Norm(kind, EPS), y, 64, F32)
        assert np.all(np.abs(y.read(np.float32) - want) <= 1e-6)


def test_nan_stays_in_its_row(hip):
    up = hip.DeviceBuffer.from_array
    x = np.ones((3, 96), np.float32)
    x[1, 5] = np.nan
    y = up(np.zeros((3, 96), np.float32))
    hip.norm_block(up(x), 96, F32, 3, 96, None, None, 0, None, 0, 0.0, None, 96, F32, hip.Norm(RMS, EPS), y, 96, F32)
    got = y.read(np.float32).reshape(3, 96)
    assert np.all(np.isnan(got[1])) and np.all(np.isfinite(got[[0, 2]]))


def test_refusals(hip):
    up = hip.DeviceBuffer.from_array
    z, small = up(np.zeros(256, np.float32)), up(np.zeros(4, np.float32))
    n = hip.Norm(RMS, EPS)

    def call(x=z, xs=64, xt=F32, M=4, N=64, post=None, gate=None, gs=0, res=None, rs=64, h=None, hs=64, ht=F32, pre=n, y=z, ys=64, yt=F32):
        hip.norm_block(x, xs, xt, M, N, post, gate, gs, res, rs, 1.0, h, hs, ht, pre, y, ys, yt)
    call()
    for match, kw in [("values", {"N": 0}), ("-1 rows", {"M": -1}), ("without an output", {"pre": None}), ("below its width", {"xs": 60}), ("dtype 4", {"xt": 4}),
                      ("residual dtype 3", {"ht": 3}), ("needs .* bytes", {"x": small}), ("needs .* bytes", {"y": small}), ("needs .* bytes", {"res": small}),
                      ("gate needs", {"gate": small}), ("gate stride 8", {"gate": z, "gs": 8}), ("norm kind 2", {"pre": hip.Norm(2, EPS)}), ("eps", {"post": hip.Norm(0, -1.0)}),
                      ("norm weights needs", {"pre": hip.Norm(0, EPS, small)}), ("normed output dtype", {"yt": 9})]:
        with pytest.raises(_abi.HipBackendError, match=match):
            call(**kw)
    big = up(np.zeros(4096, np.float32))
    with pytest.raises(_abi.HipBackendError, match="one stride"):
        call(res=big, rs=64, h=big, hs=128)
