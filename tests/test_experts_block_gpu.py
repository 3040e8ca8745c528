"""A block of experts run as a program runs it (bybylang_amd/experts.py): every step against 64 bits of what the step before left on the
device, recorded steps against eager ones bit for bit (graphs and direct replays, between other work), and no device memory taken by
any call. Bounds as in test_mx_gpu.py and test_moe_gpu.py.
"""
import numpy as np
import pytest

from bybylang_amd import _abi, synth
from mx_ref import MX4, MX8, close_mx, plan, route, rows
from paged_ref import close, norm
from test_mx_gpu import agree, expected, mx_size

pytestmark = pytest.mark.gpu
F32 = _abi.F32
U = 2.0**-24


@pytest.fixture
def gb(hip):
    from bybylang_amd import gpubackend as g
    yield g
    g.sessionRecoverQueue(g.gbHip)
    _abi.check(_abi.load().byhip_session_set_direct_replay(0))


class Block:
    def __init__(self, gb, D, F, E, k, T, seed=1, **kw):
        from bybylang_amd.experts import ExpertsBlock, random_matrix
        self.rng = synth.rng(seed)
        self.m = [random_matrix(self.rng, r, w) for r, w in ((E, D), (2 * E * F, D), (E * D, F))]
        self.gamma = self.rng.uniform(0.5, 1.5, D).astype(np.float32)
        self.bias = (0.1 * self.rng.standard_normal(E)).astype(np.float32) if kw.pop("bias", False) else None
        self.block = ExpertsBlock(*self.m, self.gamma, D, F, E, k, T, bias=self.bias, **kw)
        self.gb, self.sizes = gb, (D, F, E, k)

    def bytes(self, handle, n):
        return self.gb.sessionRead(self.gb.gbHip, handle, (n + 3) // 4).view(np.uint8)[:n]

    def floats(self, handle, *shape):
        return self.gb.sessionRead(self.gb.gbHip, handle, int(np.prod(shape))).reshape(shape)


@pytest.mark.parametrize("T", [1, 5, 70])
@pytest.mark.parametrize("kw", [dict(), dict(score=_abi.MOE_SIGMOID, bias=True, groups=4, top_groups=2, group_by=2, scale=1.5)])
@pytest.mark.parametrize("D,F,E,k", [(256, 128, 16, 4), (160, 96, 12, 2)])
def test_block_against_64_bits(gb, T, kw, D, F, E, k):
    b = Block(gb, D, F, E, k, T, seed=T + E, **kw)
    x, h = b.rng.standard_normal((T, D)).astype(np.float32), b.rng.standard_normal((T, D)).astype(np.float32)
    bx, bh, out = gb.sessionUpload(gb.gbHip, x), gb.sessionUpload(gb.gbHip, h), gb.sessionAllocScratch(gb.gbHip, T * D)
    assert b.block.encode(bx, T, bh, out)
    hv = h.astype(np.float64) + x
    close(b.floats(bh, T, D), hv, F32, 2 * U * np.abs(hv), "h")
    f = 1 / np.sqrt((hv * hv).mean(1, keepdims=True) + 1e-5)
    q = b.bytes(b.block.xq, mx_size(T, D, MX8))
    close_mx(q, norm(hv, _abi.NORM_RMS, 1e-5, b.gamma, None), 65 * U * f * b.gamma * np.abs(hv), MX8, "normed")
    xv = rows(q, T, D, MX8)
    router, up, down = (rows(b.bytes(m, mx_size(r, w, MX4)), r, w, MX4) for m, r, w in zip(b.m, (E, 2 * E * F, E * D), (D, D, F)))
    logits = b.floats(b.block.logits, T, E)
    want, slack = expected(xv, router, E, D, False, MX8, F32)
    close(logits, want, F32, slack, "logits")
    ids = b.floats(b.block.ids, T, k).view(np.int32)
    r = dict(dict(score=_abi.MOE_SOFTMAX, groups=1, top_groups=1, group_by=1, scale=1.0), **{n: v for n, v in kw.items() if n != "bias"})
    want_ids, want_w = route(logits.astype(np.float64), None if b.bias is None else b.bias.astype(np.float64), k, r["score"], r["groups"], r["top_groups"],
                             r["group_by"], True, r["scale"])
    assert np.array_equal(ids, want_ids)
    w = b.floats(b.block.shares, T, k)
    close(w, want_w, F32, (E / 64 + 16 + k + 2 * np.ptp(logits)) * U * np.abs(want_w), "weights")
    offsets, order = plan(ids, E)
    mid = b.bytes(b.block.mid, mx_size(T * k, F, MX8))
    mv = rows(mid, T * k, F, MX8)
    hidden, hs, o, os_ = np.zeros((T * k, F)), np.zeros((T * k, F)), np.zeros((T * k, D)), np.zeros((T * k, D))
    for e in range(E):
        at = np.arange(offsets[e], offsets[e + 1])
        if not at.size:
            continue
        hidden[at], hs[at] = expected(xv[order[at] // k], up.reshape(E, 2 * F, D)[e], F, D, True, MX8, MX8)
        o[order[at]], os_[order[at]] = expected(mv[at], down.reshape(E, D, F)[e], D, F, False, MX8, F32)
    agree(mid, hidden, hs, MX8, T * k, F, F)
    close(b.floats(b.block.rows, T * k, D), o, F32, os_, "rows")
    terms = o.reshape(T, k, D) * w[..., None]
    close(b.floats(out, T, D), terms.sum(1), F32, (os_.reshape(T, k, D) * np.abs(w)[..., None]).sum(1) + (k + 2) * U * np.abs(terms).sum(1), "out")


@pytest.mark.parametrize("direct", [0, 1])
@pytest.mark.parametrize("T", [3, 200])
def test_recorded(gb, direct, T):
    """A recording replayed over new inputs, with eager calls of another size (and plan) between, gives what eager calls give."""
    _abi.check(_abi.load().byhip_session_set_direct_replay(direct))
    D, F, E, k = 256, 128, 24, 3
    b = Block(gb, D, F, E, k, 200)
    bx, bh, out = gb.sessionUpload(gb.gbHip, np.zeros(T * D, np.float32)), gb.sessionUpload(gb.gbHip, np.zeros(T * D, np.float32)), gb.sessionAllocScratch(gb.gbHip, T * D)

    def put(handle, a):
        a = np.ascontiguousarray(a, np.float32)
        _abi.check(_abi.load().byhip_upload(handle.ptr, 0, a.ctypes.data, a.nbytes))
    inputs = [(b.rng.standard_normal((T, D)), b.rng.standard_normal((T, D))) for _ in range(4)]
    want = []
    for x, h in inputs:
        put(bx, x), put(bh, h)
        assert b.block.encode(bx, T, bh, out)
        want.append((b.floats(out, T, D), b.floats(bh, T, D), b.floats(b.block.ids, T, k)))
    other = [gb.sessionUpload(gb.gbHip, b.rng.standard_normal(60 * D).astype(np.float32)) for _ in range(3)]
    before = _abi.load().byhip_debug_alloc_count()
    assert gb.sessionBeginRecording(gb.gbHip)
    assert b.block.encode(bx, T, bh, out)
    assert gb.sessionEnd(gb.gbHip)
    step = gb.sessionLastRecording(gb.gbHip)
    for turn in range(2):
        for (x, h), (o, hw, ids) in zip(inputs, want):
            put(bx, x), put(bh, h)
            assert b.block.encode(other[0], 60, other[1], other[2])
            assert gb.sessionReplay(gb.gbHip, step, 1)
            assert np.array_equal(b.floats(out, T, D).view(np.uint32), o.view(np.uint32))
            assert np.array_equal(b.floats(bh, T, D), hw) and np.array_equal(b.floats(b.block.ids, T, k).view(np.int32), ids.view(np.int32))
    assert _abi.load().byhip_debug_alloc_count() == before
    gb.sessionFreeRecording(gb.gbHip, step)


def test_decoder_with_experts(gb):
    """A paged decoder's recorded steps with experts after each attention block are its eager steps."""
    from bybylang_amd import paged_decoder as p
    W, H, KV, DIM, slots = 256, 8, 2, 64, 4

    def make():
        rng = synth.rng(9)
        ws = [(p.random_weights(rng, W, H * DIM), p.random_weights(rng, W, KV * DIM), p.random_weights(rng, W, KV * DIM), p.random_weights(rng, H * DIM, W)) for _ in range(2)]
        ex = [p.ExpertsBlock(p.random_matrix(rng, 16, W), p.random_matrix(rng, 16 * 256, W), p.random_matrix(rng, 16 * W, 128), np.ones(W, np.float32), W, 128, 16, 4, 128)
              for _ in ws]
        return p.PagedDecoder(ws, [np.ones(W, np.float32)] * 3, W, H, KV, DIM, slots, 96, 128, 40, 16, experts=ex), rng
    d, rng = make()
    e, _ = make()
    prompt, counts = rng.standard_normal((90, W)), [30, 25, 34, 1]
    first = d.forward(prompt, counts)
    assert np.isfinite(first).all() and np.array_equal(first, e.forward(prompt, counts))
    plain = make()[0]
    plain.experts = [None, None]
    assert not np.array_equal(first, plain.forward(prompt, counts))
    x = rng.standard_normal((slots, W))
    for m in (d, e):
        m.set_rows([1] * slots)
        m.set_input(x)
    step = d.record()
    e.encode()
    assert np.array_equal(d.output(), e.output())
    for i in range(4):
        x = rng.standard_normal((slots, W))
        d.set_input(x), e.set_input(x)
        assert gb.sessionReplay(gb.gbHip, step, 1)
        e.encode()
        assert np.array_equal(d.output(), e.output())
    gb.sessionFreeRecording(gb.gbHip, step)
