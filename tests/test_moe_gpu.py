"""Routing, plans and experts' products on the MI355X against 64 bits (mx_ref.py).

Bounds. A softmax weight: exp's argument is rounded to 2^-24 of its size, the sum has at most E / 64 terms in a row and 6 more
levels, and a few roundings of the value: (E / 64 + 16 + 2 max|x - top|) 2^-24 of it; with the sum of the chosen another k.
A combined row of k terms: (k + 2) 2^-24 of the sum of the terms' magnitudes. Products as in test_mx_gpu.py.
"""
import numpy as np
import pytest

from bybylang_amd import _abi, synth
from mx_ref import MX4, MX8, plan, quantize, random_rows, route
from paged_ref import close, from_bits, to_bits
from test_mx_gpu import agree, expected, mx_size

pytestmark = pytest.mark.gpu
F32, F16, BF16 = _abi.F32, _abi.F16, _abi.BF16
NP = {F32: np.float32, F16: np.float16, BF16: np.uint16}
SOFT, SIG = _abi.MOE_SOFTMAX, _abi.MOE_SIGMOID
GATHER, SCATTER, GLU = _abi.MOE_GATHER, _abi.MOE_SCATTER, _abi.MOE_SWIGLU
U = 2.0**-24


def new_plan(hip, T, k, E):
    n = hip.moe_plan_bytes(T, k, E)
    buf = hip.DeviceBuffer.from_array(np.full(n + 16, 0xA5, np.uint8))
    return buf, hip.MoePlan(buf, T, k, E)


def read_plan(buf, T, k, E):
    raw = buf.read(np.uint8)
    assert np.all(raw[-16:] == 0xA5), "written past the plan"
    ints = raw[:4 * (E + 1 + T * k)].view(np.int32)
    return ints[:E + 1], ints[E + 1:]


def routed(hip, x, dt, k, score=SOFT, bias=None, groups=1, top_groups=1, group_by=1, renorm=True, scale=1.0, pad=0):
    T, E = x.shape
    wide = np.zeros((T, E + pad), x.dtype)
    wide[:, :E] = x
    up = hip.DeviceBuffer.from_array
    ids, w = up(np.full(T * k + 4, -7, np.int32)), up(np.full(T * k + 4, -7, np.float32))
    b = None if bias is None else up(bias)
    buf, p = new_plan(hip, T, k, E)
    hip.moe_route(up(wide), E + pad, dt, hip.MoeRouter(score, b, groups, top_groups, group_by, renorm, scale), p, ids, w)
    i, v = ids.read(np.int32, T * k + 4), w.read(np.float32, T * k + 4)
    assert np.all(i[T * k:] == -7) and np.all(v[T * k:] == -7)
    i, v = i[:T * k].reshape(T, k), v[:T * k].reshape(T, k)
    offsets, order = read_plan(buf, T, k, E)
    want = plan(i, E)
    assert np.array_equal(offsets, want[0]) and np.array_equal(order, want[1])
    return i, v


def check_route(hip, T, E, k, dt=F32, seed=0, bias=False, pad=0, x=None, **kw):
    g = synth.rng(900 + seed)
    x = to_bits(2 * g.standard_normal((T, E)), dt) if x is None else x
    b = (0.3 * g.standard_normal(E)).astype(np.float32) if bias else None
    got = routed(hip, x, dt, k, bias=b, pad=pad, **kw)
    a = {"score": SOFT, "groups": 1, "top_groups": 1, "group_by": 1, "renorm": True, "scale": 1.0, **kw}
    xd = from_bits(x, dt)
    ids, w = route(xd, None if b is None else b.astype(np.float64), k, a["score"], a["groups"], a["top_groups"], a["group_by"], a["renorm"], a["scale"])
    assert np.array_equal(got[0], ids)
    fine = np.where(np.isfinite(xd), xd, 0)
    reach = np.minimum(fine.max(1) - fine.min(1), 104.0)  # exp vanishes beyond
    bound = (E / 64 + 16 + k + 2 * reach[:, None]) * U
    close(got[1], w, F32, bound * np.where(np.isfinite(w), np.abs(w), 0) + 2.0**-126)


@pytest.mark.parametrize("E,k", [(1, 1), (2, 1), (2, 2), (7, 3), (8, 2), (63, 6), (64, 8), (65, 8), (100, 10), (128, 8), (130, 1), (256, 8), (257, 9), (500, 12), (512, 8), (513, 8), (1000, 7), (1024, 16)])
@pytest.mark.parametrize("T", [1, 37])
@pytest.mark.parametrize("score", [SOFT, SIG])
def test_experts(hip, E, k, T, score):
    check_route(hip, T, E, k, seed=E, score=score, renorm=E % 2 == 0, scale=1.0 + E % 3)
    check_route(hip, T, E, k, seed=E, score=score, bias=True, renorm=E % 2 == 1)


@pytest.mark.parametrize("E,k", [(70, 70), (128, 64), (200, 65), (300, 130), (1024, 200)])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_many_choices(hip, E, k, renorm, bias):
    check_route(hip, 3, E, k, seed=k, renorm=renorm, bias=bias, scale=0.5)


@pytest.mark.parametrize("E,groups,top_groups,k", [(8, 2, 1, 3), (64, 8, 3, 8), (64, 64, 9, 9), (256, 8, 4, 8), (160, 8, 3, 6), (96, 3, 2, 5), (1024, 32, 4, 8), (512, 64, 1, 8), (12, 6, 5, 4)])
@pytest.mark.parametrize("group_by", [1, 2])
@pytest.mark.parametrize("score", [SOFT, SIG])
@pytest.mark.parametrize("bias", [False, True])
def test_groups(hip, E, groups, top_groups, k, group_by, score, bias):
    check_route(hip, 23, E, k, seed=E + groups, score=score, bias=bias, groups=groups, top_groups=top_groups, group_by=group_by)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("pad", [0, 1, 4])
@pytest.mark.parametrize("bias", [False, True])
def test_types_and_strides(hip, dt, pad, bias):
    """Logits of few bits tie: the lowest index is taken."""
    check_route(hip, 50, 256, 8, dt=dt, pad=pad, bias=bias, score=SIG, seed=pad)
    g = synth.rng(4)
    x = to_bits(g.integers(-2, 3, (40, 128)).astype(np.float64), dt)
    check_route(hip, 40, 128, 9, dt=dt, pad=pad, bias=False, x=x)
    check_route(hip, 40, 128, 9, dt=dt, pad=pad, bias=False, x=x, groups=8, top_groups=3, group_by=2)


def test_keys_next_to_each_other(hip):
    """Keys that differ in the 30th bit are told apart: s + bias is ranked in 64 bits."""
    T, E, k = 8, 64, 6
    x = np.zeros((T, E), np.float32)
    x += (np.arange(E)[::-1] % 16) * np.float32(2.0**-23)
    b = np.full(E, 3.0, np.float32)
    i, _ = routed(hip, x, F32, k, score=SIG, bias=b)
    want, _ = route(x.astype(np.float64), b.astype(np.float64), k, SIG, 1, 1, 1, True, 1.0)
    assert np.array_equal(i, want)


@pytest.mark.parametrize("score", [SOFT, SIG])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("renorm", [False, True])
def test_not_finite(hip, score, bias, renorm):
    """Masked logits (-infinity), rows that are all masked, the type's lowest value, infinities and NaN: every row keeps k different experts."""
    T, E, k = 9, 40, 6
    g = synth.rng(11)
    x = g.standard_normal((T, E)).astype(np.float32)
    x[0, 5:] = -np.inf
    x[1] = -np.inf
    x[2, 3:] = np.finfo(np.float32).min
    x[3] = np.finfo(np.float32).min
    x[4, [7, 30]] = np.inf
    x[5, 9] = np.nan
    x[6] = np.nan
    x[7, ::2] = -np.inf
    check_route(hip, T, E, k, score=score, bias=bias, renorm=renorm, x=x)


@pytest.mark.parametrize("T,E,k", [(0, 4, 2), (1, 1, 1), (600, 16, 2), (4000, 60, 6), (3000, 1024, 8), (9000, 8, 2), (20000, 1, 1), (300000, 3, 1)])
def test_many_tokens(hip, T, E, k):
    g = synth.rng(T)
    x = g.standard_normal((T, E)).astype(np.float32)
    i, w = routed(hip, x, F32, k)
    want = np.argsort(-x, axis=1, kind="stable")[:, :k]
    assert np.array_equal(i, want)
    assert np.all(np.abs(w.sum(1) - 1) <= (k + 2) * U * 2)


@pytest.mark.parametrize("T,E,k", [(1, 3, 2), (200, 7, 3), (5000, 40, 4), (70000, 5, 1)])
def test_plan_of_own_ids(hip, T, E, k):
    """Ids that are nobody's are left out; the same expert twice in a row of ids counts twice."""
    g = synth.rng(T + 1)
    ids = g.integers(-1, E + 1, (T, k)).astype(np.int32)
    ids[0] = np.iinfo(np.int32).min
    if T > 1:
        ids[1], ids[2] = 1, np.iinfo(np.int32).max
    buf, p = new_plan(hip, T, k, E)
    hip.moe_plan(hip.DeviceBuffer.from_array(ids), p)
    offsets, order = read_plan(buf, T, k, E)
    want = plan(ids, E)
    assert np.array_equal(offsets, want[0]) and np.array_equal(order[:offsets[-1]], want[1])


# ── products ──


def check_product(hip, T, k, E, K, N, xf, yt, flags, seed=0, ids=None, pad=0):
    g = synth.rng(1700 + seed)
    up = hip.DeviceBuffer.from_array
    if ids is None:
        ids = np.argsort(g.standard_normal((T, E)) + 1.5 * g.standard_normal(E), axis=1)[:, :k].astype(np.int32)
    A = T * k
    glu, gather, scatter = flags & GLU, flags & GATHER, flags & SCATTER
    R = 2 * N if glu else N
    xb, xv = random_rows(g, T if gather else A, K, xf)
    wb, wv = random_rows(g, E * R, K, MX4)
    wv = wv.reshape(E, R, K)
    buf, p = new_plan(hip, T, k, E)
    hip.moe_plan(up(ids), p)
    offsets, order = plan(ids, E)
    S = N if yt in (MX8, MX4) else N + pad
    n = mx_size(A, N, yt) if yt in (MX8, MX4) else A * S * (4 if yt == F32 else 2)
    y = up(np.full(n + 16, 0xA5, np.uint8))
    hip.moe_matmul(up(xb), xf, up(wb), p, K, N, flags, y, S, yt)
    raw = y.read(np.uint8, n + 16)
    assert np.all(raw[n:] == 0xA5), "written past the end"
    want, slack, live = np.zeros((A, N)), np.zeros((A, N)), np.zeros(A, bool)
    for e in range(E):
        at = np.arange(offsets[e], offsets[e + 1])
        if at.size:
            a = order[at]
            out = a if scatter else at
            want[out], slack[out] = expected(xv[a // k if gather else at], wv[e], N, K, glu, xf, yt)
            live[out] = True
    if yt in (MX8, MX4):
        b = N if yt == MX8 else N // 2
        v, s = raw[:A * b].reshape(A, b), raw[A * b:n].reshape(A, N // 32)
        assert np.all(v[~live] == 0xA5) and np.all(s[~live] == 0xA5), "rows that are nobody's"
        raw = np.concatenate([v[live].reshape(-1), s[live].reshape(-1)])
    else:
        rows = raw[:n].reshape(A, -1)
        assert np.all(rows[~live] == 0xA5), "rows that are nobody's"
        raw = np.ascontiguousarray(rows[live]).reshape(-1)
    if live.any():
        agree(raw, want[live], slack[live], yt, int(live.sum()), N, S)


@pytest.mark.parametrize("xf", [MX8, MX4])
@pytest.mark.parametrize("T,k,E,K,N", [(1, 1, 1, 32, 32), (1, 4, 16, 512, 96), (7, 2, 5, 96, 64), (40, 8, 64, 544, 160), (100, 2, 4, 256, 128), (300, 3, 6, 384, 288), (700, 2, 3, 256, 384)])
@pytest.mark.parametrize("flags,yt", [(GATHER | GLU, MX8), (GATHER | GLU, MX4), (GATHER | GLU | SCATTER, BF16), (SCATTER, F32), (0, F16), (GATHER, F32), (GATHER, MX8), (GLU, F32)])
def test_products(hip, xf, T, k, E, K, N, flags, yt):
    check_product(hip, T, k, E, K, N, xf, yt, flags, seed=T)


@pytest.mark.parametrize("xf", [MX8, MX4])
@pytest.mark.parametrize("T,k,E,K,N", [(300, 3, 6, 256, 1056), (1000, 1, 5, 384, 1504), (90, 8, 64, 128, 1056), (2100, 2, 40, 128, 544)])
@pytest.mark.parametrize("flags,yt", [(GATHER | GLU, MX8), (GATHER | GLU, MX4), (GATHER | GLU | SCATTER, BF16), (SCATTER, F32), (0, F16), (GATHER, MX8)])
def test_products_in_tiles(hip, xf, T, k, E, K, N, flags, yt):
    """Blocks enough for moe_tiles, most experts' last one not full."""
    check_product(hip, T, k, E, K, N, xf, yt, flags, seed=T)


@pytest.mark.parametrize("flags,yt", [(GATHER | GLU, MX8), (SCATTER, F32), (GLU | SCATTER, BF16)])
def test_tiles_with_assignments_left_out(hip, flags, yt):
    g = synth.rng(3)
    check_product(hip, 500, 2, 5, 256, 1056, MX8, yt, flags, ids=g.integers(-2, 7, (500, 2)).astype(np.int32), seed=5)
    check_product(hip, 500, 2, 5, 128, 1056, MX8, yt, flags, ids=np.full((500, 2), 3, np.int32), seed=5)
    check_product(hip, 500, 2, 5, 128, 1056, MX8, yt, flags, ids=np.full((500, 2), 5, np.int32), seed=5)


@pytest.mark.parametrize("T,k,E", [(33, 2, 9), (400, 2, 4)])
@pytest.mark.parametrize("flags,yt", [(GATHER | GLU, MX8), (SCATTER, F32), (SCATTER, BF16), (GLU | SCATTER, MX4)])
def test_assignments_left_out(hip, T, k, E, flags, yt):
    g = synth.rng(2)
    ids = g.integers(-2, E + 2, (T, k)).astype(np.int32)
    check_product(hip, T, k, E, 256, 96, MX8, yt, flags, ids=ids, seed=5)
    check_product(hip, T, k, E, 256, 96, MX8, yt, flags, ids=np.full((T, k), -1, np.int32), seed=5)


@pytest.mark.parametrize("T,E", [(50, 30), (500, 12), (1000, 200)])
@pytest.mark.parametrize("flags,yt", [(GATHER | GLU, MX8), (SCATTER, F32)])
def test_all_to_one_expert(hip, T, E, flags, yt):
    """One expert gets everything (many of its units), or all but one row."""
    ids = np.full((T, 2), E - 2, np.int32)
    check_product(hip, T, 2, E, 160, 64, MX8, yt, flags, ids=ids, seed=6)
    ids[T // 2, 1] = 0
    check_product(hip, T, 2, E, 128, 64, MX8, yt, flags, ids=ids, seed=6)


@pytest.mark.parametrize("N,pad,yt,flags", [(33, 0, F32, SCATTER), (65, 3, F16, GLU), (127, 1, BF16, GATHER), (1, 0, F32, GLU), (258, 2, BF16, SCATTER)])
@pytest.mark.parametrize("T", [9, 300])
def test_odd_widths(hip, N, pad, yt, flags, T):
    check_product(hip, T, 2, 4, 256, N, MX8, yt, flags, pad=pad, seed=N)


# ── combine ──


@pytest.mark.parametrize("T,k,N,xt,rt,yt,pad", [(1, 1, 1, F32, F32, F32, 0), (5, 3, 33, F16, None, F32, 1), (17, 8, 1024, BF16, F32, BF16, 0), (3, 2, 5000, F32, BF16, F16, 4), (200, 6, 64, BF16, BF16, BF16, 0),
                                                (2, 70, 96, F32, F32, F32, 0)])
def test_combine(hip, T, k, N, xt, rt, yt, pad):
    g = synth.rng(60 + N)
    up = hip.DeviceBuffer.from_array
    E, S = max(4, k), N + pad
    x, w = to_bits(g.standard_normal((T * k, S)), xt), g.standard_normal((T, k)).astype(np.float32)
    r = None if rt is None else to_bits(g.standard_normal((T, S)), rt)
    ids = g.integers(0, E, (T, k)).astype(np.int32)
    ids[0, 0] = -1
    ids[-1, -1] = E
    xv = from_bits(x, xt)[:, :N].reshape(T, k, N)
    x = x.copy()
    x[[0, -1]] = to_bits(np.full(S, np.nan), xt)  # nobody's rows
    buf, p = new_plan(hip, T, k, E)
    y = up(np.full((T, S), 0x5A, np.uint8).repeat(4 if yt == F32 else 2).view(NP[yt]))
    hip.moe_combine(up(x), S, xt, N, p, up(ids), up(w), None if r is None else up(r), S, rt or F32, y, S, yt)
    live = ((ids >= 0) & (ids < E))[..., None]
    terms = np.where(live, xv * w[..., None], 0.0)
    res = 0 if r is None else from_bits(r, rt)[:, :N]
    got = y.read(NP[yt], T * S).reshape(T, S)
    assert np.all(np.ascontiguousarray(got[:, N:]).view(np.uint8) == 0x5A)
    close(from_bits(got[:, :N], yt), res + terms.sum(1), yt, (k + 2) * U * (np.abs(terms).sum(1) + np.abs(res)))


def test_combine_in_place(hip):
    T, k, N = 6, 2, 100
    g = synth.rng(61)
    up = hip.DeviceBuffer.from_array
    x, r = g.standard_normal((T * k, N)).astype(np.float32), g.standard_normal((T, N)).astype(np.float32)
    _, p = new_plan(hip, T, k, 4)
    y = up(r)
    hip.moe_combine(up(x), N, F32, N, p, up(np.zeros((T, k), np.int32)), up(np.full((T, k), 0.5, np.float32)), y, N, F32, y, N, F32)
    want = r.astype(np.float64) + 0.5 * x.reshape(T, k, N).astype(np.float64).sum(1)
    close(y.read(np.float32, T * N).reshape(T, N), want, F32, 4 * U * (np.abs(r) + np.abs(x.reshape(T, k, N)).sum(1)))


# ── refusals ──


def test_refusals(hip):
    up = hip.DeviceBuffer.from_array
    z, small, ints = up(np.zeros(8192, np.float32)), up(np.zeros(3, np.float32)), up(np.zeros(64, np.int32))
    buf = hip.DeviceBuffer(hip.moe_plan_bytes(4, 2, 8))
    good = hip.MoePlan(buf, 4, 2, 8)

    def rt(logits=z, stride=8, dt=F32, plan=good, ids=ints, w=z, **kw):
        hip.moe_route(logits, stride, dt, hip.MoeRouter(**kw), plan, ids, w)

    def mm(x=z, xf=MX8, w=z, plan=good, K=64, N=32, flags=0, y=z, ys=32, yt=F32):
        hip.moe_matmul(x, xf, w, plan, K, N, flags, y, ys, yt)

    def cb(x=z, xs=32, xt=F32, N=32, plan=good, ids=ints, w=z, res=None, rs=32, rd=F32, y=z, ys=32, yt=F32):
        hip.moe_combine(x, xs, xt, N, plan, ids, w, res, rs, rd, y, ys, yt)
    hip.moe_plan(ints, good)
    rt(), mm(), cb(x=up(np.zeros(512, np.float32)))
    odd = type("At", (), {"ptr": buf.ptr + 4})()
    for call, match, kw in [
            (rt, "score 2", {"score": 2}), (rt, "groups of 8 experts", {"groups": 3}), (rt, "best 0 of", {"groups": 2, "top_groups": 0}), (rt, "best 3 of", {"groups": 2, "top_groups": 3}),
            (rt, "by their 3 best", {"groups": 2, "group_by": 3}), (rt, "2 choices among 1", {"groups": 8}), (rt, "below its width", {"stride": 7}), (rt, "dtype 4", {"dt": 4}),
            (rt, "logits needs", {"logits": small}), (rt, "bias needs", {"bias": small}), (rt, "ids needs", {"ids": small}), (rt, "weights needs", {"w": small}),
            (rt, "plan needs", {"plan": hip.MoePlan(small, 4, 2, 8)}), (rt, "aligned", {"plan": hip.MoePlan(odd, 2, 2, 8)}), (rt, "a plan of", {"plan": hip.MoePlan(buf, 4, 9, 8)}),
            (rt, "a plan of", {"plan": hip.MoePlan(buf, 4, 2, 1025)}), (rt, "a plan of", {"plan": hip.MoePlan(buf, 4, 257, 1024)}), (rt, "a plan of", {"plan": hip.MoePlan(buf, -1, 2, 8)}), (rt, "a plan of", {"plan": hip.MoePlan(buf, 2**23, 2, 8)}),
            (mm, "flags 8", {"flags": 8}), (mm, "multiple of 32", {"K": 33}), (mm, "rows of a product needs", {"x": small}), (mm, "matrices .* needs", {"w": small}), (mm, "product needs", {"y": small}),
            (mm, "format 2", {"xf": BF16}), (mm, "multiple of 32", {"N": 40, "ys": 40, "yt": MX4}), (mm, "below its width", {"ys": 16}), (mm, "plan needs", {"plan": hip.MoePlan(small, 4, 2, 8)}),
            (cb, "rows of 0 values", {"N": 0}), (cb, "rows needs", {"x": small}), (cb, "residual needs", {"res": small}), (cb, "summed rows needs", {"y": small}), (cb, "ids needs", {"ids": small}),
            (cb, "weights needs", {"w": small}), (cb, "dtype 3", {"xt": 3}), (cb, "dtype 4", {"yt": 4}), (cb, "one stride", {"res": z, "rs": 64, "y": z})]:
        with pytest.raises(_abi.HipBackendError, match=match):
            call(**kw)
    with pytest.raises(ValueError, match="a plan of"):
        hip.moe_plan_bytes(4, 0, 8)


def test_no_tokens(hip):
    buf, p = new_plan(hip, 0, 2, 4)
    z = hip.DeviceBuffer.from_array(np.full(64, 7, np.float32))
    hip.moe_plan(z, p)
    assert np.all(read_plan(buf, 0, 2, 4)[0] == 0)
    hip.moe_matmul(z, MX8, hip.DeviceBuffer(4 * 32 * 17), p, 32, 32, 0, z, 32, F32)
    hip.moe_combine(z, 32, F32, 32, p, z, z, None, 0, F32, z, 32, F32)
    assert np.all(z.read(np.float32, 64) == 7)


@pytest.mark.parametrize("fill", [0, 1, 0x7F, 0xFF])
def test_buffer_without_a_plan(hip, fill):
    """A product with a buffer that no plan was made in writes rows of its own output or none, and reads its operands only."""
    for T, K, N in ((9, 64, 32), (400, 128, 2080)):
        check_no_plan(hip, fill, T, K, N)


def check_no_plan(hip, fill, T, K, N):
    k, E = 2, 4
    up = hip.DeviceBuffer.from_array
    buf = up(np.full(hip.moe_plan_bytes(T, k, E), fill, np.uint8))
    p = hip.MoePlan(buf, T, k, E)
    y = up(np.full(T * k * N + 64, 7, np.float32))
    x, w = up(np.zeros(mx_size(T * k, K, MX8), np.uint8)), up(np.zeros(mx_size(E * N, K, MX4), np.uint8))
    for flags in (0, GATHER, SCATTER | GATHER):
        hip.moe_matmul(x, MX8, w, p, K, N, flags, y, N, F32)
        got = y.read(np.float32)
        assert np.all((got == 0) | (got == 7)) and np.all(got[T * k * N:] == 7)


def test_quantized_rows_through_experts(hip):
    """Rows quantised on the device, routed, multiplied, brought back to 8 bits, multiplied again and summed: each step against 64 bits of what the
    step before left."""
    T, E, k, D, F = 45, 12, 3, 256, 160
    g = synth.rng(70)
    up = hip.DeviceBuffer.from_array
    x = g.standard_normal((T, D)).astype(np.float32)
    xq, mid, dn = hip.DeviceBuffer(mx_size(T, D, MX8)), hip.DeviceBuffer(mx_size(T * k, F, MX8)), hip.DeviceBuffer(T * k * D * 4)
    ids, w, y = hip.DeviceBuffer(T * k * 4), hip.DeviceBuffer(T * k * 4), hip.DeviceBuffer(T * D * 4)
    w1, w2 = random_rows(g, E * 2 * F, D, MX4), random_rows(g, E * D, F, MX4)
    buf, p = new_plan(hip, T, k, E)
    b1, b2, bx = up(w1[0]), up(w2[0]), up(x)
    hip.mx_quantize(bx, D, F32, T, D, xq, MX8)
    hip.moe_route(up(g.standard_normal((T, E)).astype(np.float32)), E, F32, hip.MoeRouter(), p, ids, w)
    hip.moe_matmul(xq, MX8, b1, p, D, F, GATHER | GLU, mid, F, MX8)
    hip.moe_matmul(mid, MX8, b2, p, F, D, SCATTER, dn, D, F32)
    hip.moe_combine(dn, D, F32, D, p, ids, w, bx, D, F32, y, D, F32)
    from mx_ref import rows
    xv = rows(xq.read(np.uint8), T, D, MX8)
    assert np.array_equal(xv, quantize(x, MX8)[1])
    chosen = ids.read(np.int32).reshape(T, k)
    offsets, order = plan(chosen, E)
    h = mid.read(np.uint8)
    hv = rows(h, T * k, F, MX8)
    wv1, wv2 = w1[1].reshape(E, 2 * F, D), w2[1].reshape(E, D, F)
    want, slack = np.zeros((T * k, F)), np.zeros((T * k, F))
    out, oslack = np.zeros((T * k, D)), np.zeros((T * k, D))
    for e in range(E):
        at = np.arange(offsets[e], offsets[e + 1])
        if not at.size:
            continue
        want[at], slack[at] = expected(xv[order[at] // k], wv1[e], F, D, True, MX8, MX8)
        out[order[at]], oslack[order[at]] = expected(hv[at], wv2[e], D, F, False, MX8, F32)
    agree(h, want, slack, MX8, T * k, F, F)
    close(dn.read(np.float32).reshape(T * k, D), out, F32, oslack)
    terms = out.reshape(T, k, D) * w.read(np.float32).reshape(T, k, 1)
    aw = np.abs(w.read(np.float32)).reshape(T, k, 1)
    close(y.read(np.float32).reshape(T, D), x + terms.sum(1), F32, (oslack.reshape(T, k, D) * aw).sum(1) + (k + 3) * U * (np.abs(terms).sum(1) + np.abs(x)))
