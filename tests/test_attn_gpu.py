"""byhip_paged_attention against attention in 64 bits, through device.paged_attention.

Bounds. A score is a sum of D products in fp32 (or of products of 16-bit terms that hold 22 bits and more of an fp32
query), rounded D times in some order: errors that add up like a random walk, taken at twice its deviation, 2
sqrt(D) 2^-24 of sum |q_d k_d| scale. The exponential's argument and value, the cap's tanh (2^-22 of the cap) and the bias
add 4e-6 for every weight that counts, and the sums over L keys sqrt(L) 2^-22. A weight off by a share e moves
the output by at most e (mean |v| + |out|). With 16-bit queries and output a weight is also rounded to the cache's dtype: half a
unit of it in mean |v|, and 2^-25 a key where fp16 ends.
"""
import numpy as np
import pytest

from bybylang_amd import _abi, synth
from paged_ref import UNIT, attention, close, from_bits, paged, to_bits

pytestmark = pytest.mark.gpu
F32, F16, BF16 = _abi.F32, _abi.F16, _abi.BF16
NP = {F32: np.float32, F16: np.float16, BF16: np.uint16}


class Case:
    """A cache with its sequences on the device, and the expected rows."""

    def __init__(self, hip, lens, new, H, Hk, D, page, ct=F16, qt=None, ot=None, pad=0, cap=0.0, window=0, slopes=False, prefix=None,
                 seed=0, sharp=1.5, scale=None, cols=0):
        self.hip, self.lens, self.new, self.H, self.Hk, self.D, self.page, self.ct = hip, lens, new, H, Hk, D, page, ct
        self.qt, self.ot = ct if qt is None else qt, ct if ot is None else ot
        g = self.g = synth.rng(6300 + seed)
        self.T, self.W = sum(new), H * D + pad
        self.pages = sum(-(-n // page) for n in lens) + 2
        self.table = paged(g, lens, page, self.pages, cols)
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.q = to_bits(sharp * g.standard_normal((max(self.T, 1), self.W)), self.qt)
        self.kv = [to_bits(g.standard_normal((self.pages, Hk, page, D)), ct) for _ in range(2)]
        self.scale = D ** -0.5 if scale is None else scale
        self.cap, self.window = cap, window
        self.slopes = (2.0 ** (-8.0 * np.arange(1, H + 1) / H)).astype(np.float32) if slopes else None
        self.prefix = None if prefix is None else np.array(prefix, np.int32)

    def run(self):
        hip, up = self.hip, self.hip.DeviceBuffer.from_array
        self.keep = [up(a) for a in (self.q, self.kv[0], self.kv[1], self.table, self.starts, np.array(self.lens, np.int32))]
        q, k, v, t, s, n = self.keep
        opt = [None if a is None else up(a) for a in (self.slopes, self.prefix)]
        cache = hip.KvCache(k, v, self.ct, self.pages, self.page, self.Hk, self.D)
        batch = hip.KvBatch(t, self.table.shape[1], s, n, len(self.lens), self.T)
        fill = to_bits(np.full((max(self.T, 1), self.W), 77.0), self.ot)
        out = up(fill)
        hip.paged_attention(q, self.W, self.qt, self.H, hip.Attn(self.scale, self.cap, self.window, *opt), cache, batch, out, self.W, self.ot)
        got = out.read(NP[self.ot], fill.size).reshape(fill.shape)
        assert np.array_equal(got[:, self.H * self.D:], fill[:, self.H * self.D:]), "columns between rows were written"
        return from_bits(got, self.ot)[:, :self.H * self.D].reshape(-1, self.H, self.D)

    def sequence(self, b):
        L = self.lens[b]
        at = np.arange(L)
        pg = self.table[b, at // self.page]
        there = (pg >= 0) & (pg < self.pages)
        k, v = (from_bits(a, self.ct)[np.where(there, pg, 0), :, at % self.page] for a in self.kv)
        return k, v, there

    def check(self, got=None):
        got = self.run() if got is None else got
        q = from_bits(self.q, self.qt)[:, :self.H * self.D].reshape(-1, self.H, self.D)
        for b, n in enumerate(self.new):
            if n == 0:
                continue
            t = slice(self.starts[b], self.starts[b] + n)
            k, v, there = self.sequence(b)
            out, mean, size, flat = attention(q[t], k, v, float(np.float32(self.scale)), self.cap, self.window, self.slopes,
                                              0 if self.prefix is None else int(self.prefix[b]), there)
            share = 2 * np.sqrt(self.D) * 2.0**-24 * size + 4e-6 + self.cap * 2.0**-22 + np.sqrt(self.lens[b]) * 2.0**-22
            with np.errstate(invalid="ignore"):
                slack = share * (mean + np.abs(out))
                if F32 not in (self.qt, self.ot):
                    slack = slack + UNIT[self.ct] * mean + (2.0**-25 * flat if self.ct == F16 else 0)
            close(got[t], out, self.ot, slack, f"sequence {b}")
        return got


TYPES = [(F16, F16, F16), (BF16, BF16, BF16), (F16, F32, F32), (BF16, F32, F32), (F16, F32, F16), (BF16, BF16, F32)]


@pytest.mark.parametrize("ct,qt,ot", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256, 80, 40, 8])
def test_types_and_heads(hip, ct, qt, ot, D):
    Case(hip, [70, 1, 33, 200], [1, 1, 33, 50], 8, 2, D, 16, ct, qt, ot, seed=D + ct).check()


@pytest.mark.parametrize("D", [1, 7, 20, 90, 260, 600])
def test_heads_of_other_sizes(hip, D):
    Case(hip, [40, 9], [3, 9], 4, 2, D, 8, F16, F32, F32, seed=D).check()


@pytest.mark.parametrize("D", [8, 72, 80, 96, 104, 136, 200])
@pytest.mark.parametrize("ct,qt", [(F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)])
def test_heads_that_do_not_fill_their_tiles(hip, D, ct, qt):
    """Prompts, chunks and single tokens of heads between the sizes that the kernels on matrix instructions are made for."""
    Case(hip, [130, 300, 77], [130, 50, 1], 6, 2, D, 16, ct, qt, qt, seed=D).check()


@pytest.mark.parametrize("H,Hk", [(1, 1), (5, 1), (7, 7), (12, 4), (16, 1), (40, 2), (33, 1)])
def test_groups(hip, H, Hk):
    Case(hip, [130, 65], [1, 40], H, Hk, 64, 16, BF16, seed=H).check()


@pytest.mark.parametrize("L", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000])
@pytest.mark.parametrize("ct,qt", [(F16, F16), (BF16, F32)])
def test_lengths(hip, L, ct, qt):
    """One token, and the whole sequence at once, as one batch and each alone."""
    Case(hip, [L, L], [1, min(L, 150)], 4, 2, 128, 16, ct, qt, qt, seed=L).check()
    Case(hip, [L], [1], 4, 2, 128, 16, ct, qt, qt, seed=L + 1).check()
    Case(hip, [L], [min(L, 70)], 2, 2, 64, 16, ct, qt, qt, seed=L + 2).check()


@pytest.mark.parametrize("page", [1, 3, 16, 64, 100, 128, 1024])
@pytest.mark.parametrize("ct,qt", [(F16, F32), (BF16, BF16)])
def test_page_sizes(hip, page, ct, qt):
    Case(hip, [333, 64, 5], [1, 64, 4], 4, 1, 64, page, ct, qt, qt, seed=page, cols=2).check()


def test_empty_sequences_and_rows(hip):
    Case(hip, [0, 10, 5, 0, 64], [0, 0, 5, 0, 1], 4, 2, 64, 16, seed=1).check()
    c = Case(hip, [3, 9], [3, 2], 2, 1, 64, 16, seed=2)
    c.lens = [2, 9]  # three rows, two tokens: the first row has position -1 and sees nothing
    got = c.check()
    assert np.all(got[0] == 0)
    c = Case(hip, [4], [2], 2, 1, 64, 4, seed=3)
    c.table[:] = -1  # no page exists
    assert np.all(c.run() == 0)
    c.table[:] = c.pages
    assert np.all(c.run() == 0)


def test_rows_outside_the_starts_stay(hip):
    c = Case(hip, [9], [3], 2, 1, 64, 16, seed=4)
    c.T = 5
    c.q = to_bits(np.ones((5, c.W)), F16)
    assert np.all(c.run()[3:] == 77)


MASKS = [dict(window=1), dict(window=20), dict(window=64), dict(cap=5.0), dict(slopes=True), dict(prefix=[0, 40, 90]), dict(prefix=[500, 1, 70], window=16),
         dict(cap=20.0, window=33, slopes=True, prefix=[10, 60, 5]), dict(cap=30.0, slopes=True), dict(window=1000, prefix=[3, 3, 3])]


@pytest.mark.parametrize("new", [[1, 2, 1], [1, 60, 40]])
def test_sequences_with_rows_past_the_calls_are_left_out(hip, new):
    """`rows` below the last start: the sequence whose rows pass it keeps its outputs as they were, the others have theirs."""
    c = Case(hip, [90, 70, 80], new, 4, 2, 64, 16, F16, F32, F32)
    up = hip.DeviceBuffer.from_array
    bufs = [up(a) for a in (c.q, c.kv[0], c.kv[1], c.table, c.starts, np.array(c.lens, np.int32))]
    q, k, v, t, s, n = bufs
    out = up(np.full((c.T, c.W), 77.0, np.float32))  # room for all rows; the call is told of fewer
    rows = int(c.starts[2])
    hip.paged_attention(q, c.W, F32, 4, hip.Attn(c.scale), hip.KvCache(k, v, F16, c.pages, 16, 2, 64),
                        hip.KvBatch(t, c.table.shape[1], s, n, 3, rows), out, c.W, F32)
    got = out.read(np.float32, c.T * c.W).reshape(c.T, 4, 64)
    assert np.all(got[rows:] == 77.0)
    c.new = new[:2] + [0]
    c.check(got.astype(np.float64))


@pytest.mark.parametrize("kw", MASKS, ids=[",".join(k) + str(i) for i, k in enumerate(MASKS)])
@pytest.mark.parametrize("ct,qt", [(F16, F16), (F16, F32), (BF16, F32)])
def test_masks_caps_and_biases(hip, kw, ct, qt):
    Case(hip, [300, 140, 77], [1, 140, 30], 4, 2, 128, 16, ct, qt, qt, seed=5, **kw).check()
    Case(hip, [300, 200, 170], [1, 1, 1], 4, 2, 64, 32, ct, qt, qt, seed=6, **kw).check()


def test_strided_rows_and_sharp_scores(hip):
    Case(hip, [200, 90], [60, 1], 4, 2, 128, 16, F16, pad=8, seed=7, sharp=20.0).check()
    Case(hip, [200, 90], [60, 1], 4, 2, 128, 16, BF16, F32, F32, pad=4, seed=8, sharp=20.0).check()
    Case(hip, [200, 90], [60, 1], 4, 2, 64, 16, F16, F32, F32, pad=3, seed=9, scale=-0.3).check()


@pytest.mark.parametrize("ct,qt", [(F16, F16), (BF16, F32)])
def test_long_contexts(hip, ct, qt):
    """One row and a few rows over a length that is split between blocks."""
    Case(hip, [40000, 12345], [1, 1], 4, 1, 128, 64, ct, qt, qt, seed=10).check()
    Case(hip, [20011], [9], 8, 2, 64, 16, ct, qt, qt, seed=11).check()
    Case(hip, [9000, 7000], [33, 1], 4, 2, 128, 16, ct, qt, qt, seed=12, window=5000, prefix=[100, 0]).check()


@pytest.mark.parametrize("new", [1, 40, 200])
@pytest.mark.parametrize("poison", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("ct,qt", [(F16, F16), (F16, F32), (BF16, BF16)])
def test_hidden_keys_have_no_influence(hip, new, poison, ct, qt):
    """NaN and infinities in pages past the length, before the window and after a row's position."""
    c = Case(hip, [230], [new], 4, 2, 128, 32, ct, qt, qt, window=100, seed=13)
    want = c.run()
    bad = to_bits(np.array([poison]), ct)[0]
    used = np.zeros((c.pages, c.page), bool)
    first = max(0, 230 - new - 99)
    at = np.arange(first, 230)
    used[c.table[0, at // c.page], at % c.page] = True
    for a in c.kv:
        a[np.broadcast_to(~used[:, None, :], a.shape[:3])] = bad
    got = c.run()
    assert np.array_equal(got, want)
    if new > 1:  # the last key is seen by the last row alone
        for which in (0, 1):
            keep = c.kv[which].copy()
            c.kv[which][c.table[0, 229 // c.page], :, 229 % c.page] = bad
            got = c.run()
            assert np.array_equal(got[:-1], want[:-1]), "rows before a key read it"
            c.kv[which] = keep


def test_seen_infinities_and_nans_are_those_of_the_formula(hip):
    for new in (1, 20):
        for which, val in ((0, np.nan), (1, np.nan), (1, np.inf)):
            c = Case(hip, [60], [new], 2, 1, 64, 16, F16, F32, F32, seed=14)
            c.kv[which][c.table[0, 45 // 16], :, 45 % 16] = to_bits(np.array([val]), F16)[0]
            c.check()


def test_equal_runs_and_batches(hip):
    """The same bits again, and a sequence's rows do not depend on what else is in the batch's values."""
    c = Case(hip, [3000, 500, 64], [1, 30, 64], 8, 2, 128, 16, F16, seed=15)
    a, b = c.run(), c.run()
    assert np.array_equal(a, b)
    c.q[:31] = to_bits(np.zeros((31, c.W)), F16)
    assert np.array_equal(c.run()[31:], a[31:])


@pytest.mark.parametrize("ct", [F16, BF16])
def test_rows_beside_long_tables(hip, ct):
    """Tables with room for many keys, whatever the sequences hold: 4 to 24 rows per key head and single tokens."""
    Case(hip, [300, 90, 17, 200, 1000], [12, 1, 8, 2, 9], 4, 2, 64, 16, ct, ct, ct, cols=4000).check()
    Case(hip, [300], [11], 4, 2, 64, 16, ct, ct, ct, cols=16000).check()


def test_cache_past_4_gib(hip):
    g = synth.rng(6400)
    Hk, page, D, pages = 8, 64, 128, 34000  # 4.46 GB each of keys and values
    bytes_of = Hk * page * D * 2
    bk, bv = hip.DeviceBuffer(pages * bytes_of), hip.DeviceBuffer(pages * bytes_of)
    ids = [33999, 2, 33000, 17]
    kv = [to_bits(g.standard_normal((4, Hk, page, D)), F16) for _ in range(2)]
    for buf, a in ((bk, kv[0]), (bv, kv[1])):
        for i, p in enumerate(ids):
            buf.upload(a[i], p * bytes_of)
    up = hip.DeviceBuffer.from_array
    for n in (1, 80):
        L = 250
        q = to_bits(1.5 * g.standard_normal((n, 16 * D)), F16)
        out = hip.DeviceBuffer(n * 16 * D * 2)
        batch = hip.KvBatch(up(np.array(ids, np.int32)), 4, up(np.array([0, n], np.int32)), up(np.array([L], np.int32)), 1, n)
        bq = up(q)
        hip.paged_attention(bq, 16 * D, F16, 16, hip.Attn(D ** -0.5), hip.KvCache(bk, bv, F16, pages, page, Hk, D), batch, out, 16 * D, F16)
        got = from_bits(out.read(np.float16, n * 16 * D), F16).reshape(n, 16, D)
        k, v = (from_bits(a, F16).transpose(0, 2, 1, 3).reshape(-1, Hk, D)[:L] for a in kv)
        want, mean, size, flat = attention(from_bits(q, F16).reshape(n, 16, D), k, v, float(np.float32(D ** -0.5)), 0, 0, None, 0)
        share = 2 * np.sqrt(D) * 2.0**-24 * size + 4e-6 + np.sqrt(L) * 2.0**-22
        close(got, want, F16, share * (mean + np.abs(want)) + UNIT[F16] * mean + 2.0**-25 * flat)


def test_refusals(hip):
    up = hip.DeviceBuffer.from_array
    z, small, ints = up(np.zeros(4096, np.float32)), up(np.zeros(4, np.float32)), up(np.zeros(64, np.int32))

    def call(heads=2, q=z, qs=128, qt=F16, attn=None, cache=None, batch=None, out=z, os=128, ot=F16):
        hip.paged_attention(q, qs, qt, heads, attn or hip.Attn(0.1), cache or hip.KvCache(z, z, F16, 2, 4, 2, 64),
                            batch or hip.KvBatch(ints, 4, ints, ints, 2, 4), out, os, ot)
    call()
    E, U = _abi.HipBackendError, _abi.HipUnsupported
    for err, match, kw in [
            (E, "3 heads over 2", {"heads": 3}), (E, "0 heads", {"heads": 0}), (U, "cache's dtype", {"qt": BF16}), (E, "queries dtype 3", {"qt": 3}),
            (E, "output dtype 5", {"ot": 5}), (E, "below its width", {"qs": 127}), (E, "below its width", {"os": 100}), (E, "queries needs", {"q": small}),
            (E, "output needs", {"out": small}), (E, "softcap", {"attn": hip.Attn(0.1, -1.0)}), (E, "softcap", {"attn": hip.Attn(0.1, float("nan"))}),
            (E, "slopes needs", {"attn": hip.Attn(0.1, slopes=up(np.zeros(1, np.float32)))}), (E, "prefix lengths needs", {"attn": hip.Attn(0.1, prefix=up(np.zeros(1, np.int32)))}),
            (U, "fp16 or bf16", {"cache": hip.KvCache(z, z, F32, 2, 4, 2, 64)}), (E, "cache values needs", {"cache": hip.KvCache(z, small, F16, 2, 4, 2, 64)}),
            (U, "heads of 4000", {"cache": hip.KvCache(z, z, F16, 1, 1, 1, 4000), "heads": 1, "qs": 4000, "os": 4000, "batch": hip.KvBatch(ints, 4, ints, ints, 2, 1)}),
            (E, "pages each", {"batch": hip.KvBatch(ints, 0, ints, ints, 2, 4)}), (E, "lengths needs", {"batch": hip.KvBatch(ints, 1, ints, small, 8, 4)})]:
        with pytest.raises(err, match=match):
            call(**kw)
    _abi.load().byhip_fault_inject(1)
    with pytest.raises(E, match="injected fault"):
        call()
