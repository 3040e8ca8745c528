"""Rows whose byhip_cache_grow was refused: they have no position, so nothing of what the caches hold changes, whoever shares
the pages, and the sequences beside them go on as if those rows were not there."""
import numpy as np
import pytest

from bybylang_amd import _abi, synth
from paged_ref import attention, close, from_bits, to_bits
from test_paged_decoder_gpu import SLOTS, WIDTH, gb, make  # noqa: F401

pytestmark = pytest.mark.gpu
F32, F16 = _abi.F32, _abi.F16


class Small:
    """A pool of 16-token pages and its batch arrays, with what the last grows got."""

    def __init__(self, hip, lens, pages, cols, D=64, Hk=1, seed=0):
        g = self.g = synth.rng(8300 + seed)
        self.hip, self.D, self.Hk, self.pages, self.cols, self.slots = hip, D, Hk, pages, cols, len(lens)
        up = self.up = hip.DeviceBuffer.from_array
        self.kv = [to_bits(g.standard_normal((pages, Hk, 16, D)), F16) for _ in range(2)]
        self.table, at = np.full((len(lens), cols), -1, np.int32), 0
        for r, n in enumerate(lens):
            need = -(-n // 16)
            self.table[r, :need] = range(at, at + need)
            at += need
        refs = np.zeros(pages, np.int32)
        refs[:at] = 1
        self.bk, self.bv, self.bt, self.br = up(self.kv[0]), up(self.kv[1]), up(self.table), up(refs)
        self.bl, self.bs, self.bg = up(np.array(lens, np.int32)), up(np.zeros(4, np.int32)), up(np.full(len(lens), 9, np.int32))
        self.cache = hip.KvCache(self.bk, self.bv, F16, pages, 16, Hk, D)
        self.pool = hip.KvPool([self.cache], self.br, self.bt, cols, self.bl, len(lens), self.bs, self.bg)

    def ints(self, v):
        return self.up(np.array(v, np.int32))

    def grow(self, rows, add):
        self.hip.cache_grow(self.pool, self.ints(rows), self.ints(add), len(rows))

    def caches(self):
        return self.bk.read(np.uint16), self.bv.read(np.uint16)

    def append_and_attend(self, new, H=2, dtype=F32):
        """Random rows through rope_append (no rotation) and paged_attention; (q, k, v, rotated queries, outputs)."""
        T, D, Hk = sum(new), self.D, self.Hk
        q, k, v = (self.g.standard_normal((T, n * D)).astype(np.float32) for n in (H, Hk, Hk))
        out, rot = self.up(np.full((T, H * D), 5, np.float32)), self.up(np.full((T, H * D), 7, np.float32))
        starts = self.up(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
        batch = self.hip.KvBatch(self.bt, self.cols, starts, self.bl, self.slots, T, self.bg)
        self.hip.rope_append(self.up(q), H * D, self.up(k), Hk * D, self.up(v), Hk * D, F32, H, None, self.cache, batch, rot, H * D, F32)
        self.hip.paged_attention(self.up(q), H * D, dtype, H, self.hip.Attn(D ** -0.5), self.cache, batch, out, H * D, F32)
        return q, k, v, rot.read(np.float32).reshape(T, -1), out.read(np.float32).reshape(T, -1)


def test_what_grows_got(hip):
    p = Small(hip, [17, 5, 0, 30, 32, 3], 10, 3)
    p.grow([0, 1, 2, 3, 4, 5], [15, 12, 1, 0, 17, -2])  # into their pages; a page; a page; nothing asked; past the table; shrinks
    assert p.bg.read(np.int32).tolist() == [15, 12, 1, 0, 0, 0]
    p.grow([3, 5, 3, 9], [2, 2, 2, 1])   # the third names a slot twice, the fourth does not exist
    assert p.bg.read(np.int32).tolist() == [15, 12, 1, 2, 0, 2]
    assert p.bs.read(np.int32)[:2].tolist() == [1, 2]
    p.grow([0, 1, 2], [16, 40, 1])       # no page is free; past the table; nothing after the first that does not fit
    assert p.bg.read(np.int32)[:3].tolist() == [0, 0, 0]


@pytest.mark.parametrize("D", [64, 20])  # the kernels on matrix instructions; the general one
@pytest.mark.parametrize("new", [1, 5, 60])
def test_sharers_keep_their_pages(hip, D, new):
    """Slot 1 shares slot 0's 17 tokens; no page is free, so both are refused a copy of the page they would append to. Slot 2
    has room in its own page."""
    p = Small(hip, [17, 0, 3], 3, 8, D, seed=D + new)
    hip.cache_fork(p.pool, p.ints([0]), p.ints([1]), 1)
    p.grow([0, 1, 2], [new, new, 0])
    p.grow([2], [1])
    assert p.bg.read(np.int32).tolist() == [0, 0, 1]
    assert p.bl.read(np.int32).tolist() == [17, 17, 4]
    q, k, v, rot, out = p.append_and_attend([new, new, 1])
    got = p.caches()
    for a, b, x in zip(got, p.kv, (k, v)):
        want = b.view(np.uint16).copy()
        want[2, 0, 3] = to_bits(x[-1], F16).view(np.uint16)
        assert np.array_equal(a.reshape(want.shape), want)
    assert np.all(rot[:-1] == 7) and np.array_equal(rot[-1], q[-1])
    assert np.all(out[:-1] == 0)
    kv = [from_bits(a.view(np.float16).reshape(b.shape)[2, :, :4].transpose(1, 0, 2), F16) for a, b in zip(got, p.kv)]
    want, mean, size, _ = attention(q[-1:].astype(np.float64).reshape(1, 2, D), kv[0], kv[1], float(np.float32(D ** -0.5)), 0, 0, None, 0)
    close(out[-1:].reshape(1, 2, D), want, F32, (2 * np.sqrt(D) * 2.0**-24 * size + 5e-6) * (mean + np.abs(want)))


def test_more_rows_than_were_granted(hip):
    """Three rows after a grow of two: they would begin at a token that is there already."""
    p = Small(hip, [10, 20], 4, 3)
    p.grow([0, 1], [2, 2])
    before = p.caches()
    _, _, _, _, out = p.append_and_attend([3, 2])
    after = p.caches()
    for a, b in zip(before, after):
        a, b = a.reshape(4, 16, 64), b.reshape(4, 16, 64)
        assert np.array_equal(a[0], b[0]) and not np.array_equal(a[2, 4:6], b[2, 4:6])
    assert np.all(out[:3] == 0) and np.all(out[3:] != 0)


@pytest.mark.parametrize("new", [1, 20])
def test_many_sequences(hip, new):
    """More sequences than one launch counts, every third one refused."""
    B, D = 1100, 64
    g = synth.rng(8390)
    up = hip.DeviceBuffer.from_array
    kv = [to_bits(g.standard_normal((2 * B, 1, 16, D)), F16) for _ in range(2)]
    got = np.where(np.arange(B) % 3 == 0, new - 1, new).astype(np.int32)
    lens = np.full(B, 24, np.int32)
    q = g.standard_normal((B * new, D)).astype(np.float32)
    out, rot, both = up(np.full(q.shape, 5, np.float32)), up(np.full(q.shape, 7, np.float32)), [up(a) for a in kv]
    starts, table = up((np.arange(B + 1) * new).astype(np.int32)), up(np.arange(2 * B, dtype=np.int32))
    cache = hip.KvCache(*both, F16, 2 * B, 16, 1, D)
    batch = hip.KvBatch(table, 2, starts, up(lens), B, B * new, up(got))
    qk = up(q)
    hip.paged_attention(qk, D, F32, 1, hip.Attn(D ** -0.5), cache, batch, out, D, F32)
    y = out.read(np.float32).reshape(B, new, D)
    full = hip.KvBatch(table, 2, starts, up(lens), B, B * new)
    hip.paged_attention(qk, D, F32, 1, hip.Attn(D ** -0.5), cache, full, out, D, F32)
    z = out.read(np.float32).reshape(B, new, D)
    assert np.all(y[::3] == 0) and np.all(z != 0)
    keep = np.arange(B) % 3 != 0
    assert np.all(np.abs(y[keep] - z[keep]) <= 4e-6 * (1 + np.abs(z[keep])))  # parts may be cut elsewhere
    hip.rope_append(qk, D, qk, D, qk, D, F32, 1, None, cache, batch, rot, D, F32)
    r = rot.read(np.float32).reshape(B, new, D)
    assert np.all(r[::3] == 7) and np.array_equal(r[keep], q.reshape(B, new, D)[keep])
    for buf, was in zip(both, kv):
        now = buf.read(np.float16).reshape(B, 32, D)
        want = was.reshape(B, 32, D).copy()
        want[keep, 24 - new:24] = q.reshape(B, new, D)[keep].astype(np.float16)
        assert np.array_equal(now.view(np.uint16), want.view(np.uint16))


def test_short_arrays_are_refused(hip):
    p = Small(hip, [4, 4, 4], 6, 2)
    small = p.ints([0, 0])
    pool = hip.KvPool([p.cache], p.br, p.bt, 2, p.bl, 3, p.bs, small)
    with pytest.raises(_abi.HipBackendError, match="granted tokens needs 12"):
        hip.cache_grow(pool, p.ints([0]), p.ints([1]), 1)
    z = p.up(np.zeros(512, np.float32))
    batch = hip.KvBatch(p.bt, 2, p.ints([0, 1, 2, 3]), p.bl, 3, 3, small)
    with pytest.raises(_abi.HipBackendError, match="granted tokens needs 12"):
        hip.paged_attention(z, 64, F32, 1, hip.Attn(0.1), p.cache, batch, z, 64, F32)


def cache_bytes(gb, d):  # noqa: F811
    n = d.caches[0].value
    halves = n.pages * n.kv_heads * n.page_size * n.head_dim
    return [gb.sessionRead(gb.gbHip, b, halves // 2).view(np.uint16).reshape(n.pages, -1) for c in d.caches for b in c.keep[:2]]


def test_decoder_without_free_pages(gb):  # noqa: F811
    """Slot 2 forks slot 1 inside a page; then no page is free for the copies: neither writes into the page they share, and
    slot 0, which has room, goes on as in a pool that is large enough. The two runs' steps have other numbers of rows, so a
    product may differ in its last bits and a cached value be rounded the other way: 2^-10 of it, twice for two layers."""
    x = synth.rng(30).standard_normal((40, WIDTH)).astype(np.float32)
    got = []
    for pages in (4, 80):
        d, _, _ = make(gb, layers=2, pages=pages)
        d.forward(x[:2 + 19], [2, 19, 0, 0, 0, 0])  # a page and 2
        d.fork([1], [2])
        if pages == 4:
            d.forward(x[21:22], [0, 0, 0, 1, 0, 0])  # the last one
            before = cache_bytes(gb, d)
            held = gb.sessionRead(gb.gbHip, d.table, SLOTS * d.stride).view(np.int32).reshape(SLOTS, -1)
            y = d.forward(x[22:26], [1, 1, 1, 0, 0, 1])
            assert d.granted().tolist() == [1, 0, 0, 0, 0, 0] and d.refused() == 3
            assert d.lengths().tolist() == [3, 19, 19, 1, 0, 0]
            for a, b in zip(before, cache_bytes(gb, d)):
                for r in (1, 2, 3):
                    for page in held[r][held[r] >= 0]:
                        assert np.array_equal(a[page], b[page]), f"slot {r}'s page {page}"
            assert np.all(np.isfinite(y))
            d.free([3])  # now there is a page for one of the two, and the other then has the old one to itself
            z = d.forward(x[26:28], [0, 1, 1, 0, 0, 0])
            assert d.granted().tolist()[1:3] == [1, 1] and d.lengths().tolist()[1:3] == [20, 20]
        else:
            y = d.forward(x[22:23], [1, 0, 0, 0, 0, 0])
            z = d.forward(x[26:28], [0, 1, 1, 0, 0, 0])
        got.append((y[0], z))
    for a, b in zip(*got):
        assert np.all(np.abs(a - b) <= 2.0**-9 * (1 + np.abs(b)))


@pytest.mark.parametrize("direct", [False, True], ids=["graph", "direct"])
def test_replays_past_the_longest_sequence(gb, direct):  # noqa: F811
    _abi.check(_abi.load().byhip_session_set_direct_replay(int(direct)))
    d, _, _ = make(gb, layers=2)
    rng = synth.rng(31)
    d.forward(rng.standard_normal((200, WIDTH)), [157, 0, 33, 0, 10, 0])  # 160 is the longest
    d.set_rows([1, 0, 1, 0, 1, 0])
    d.set_input(rng.standard_normal((3, WIDTH)))
    step = d.record()
    while d.lengths()[0] < 160:
        assert gb.sessionReplay(gb.gbHip, step, 1)
    n = d.lengths()
    full = gb.sessionRead(gb.gbHip, d.table, SLOTS * d.stride).view(np.int32).reshape(SLOTS, -1)[0]
    before = cache_bytes(gb, d)
    for k in range(1, 4):
        d.set_input(rng.standard_normal((3, WIDTH)))
        assert gb.sessionReplay(gb.gbHip, step, 1)
        assert d.lengths().tolist() == [160, 0, n[2] + k, 0, n[4] + k, 0]
        assert d.granted().tolist() == [0, 0, 1, 0, 1, 0]
        for a, b in zip(before, cache_bytes(gb, d)):
            assert np.array_equal(a[full], b[full])
    assert d.refused() == 3
    gb.sessionFreeRecording(gb.gbHip, step)
