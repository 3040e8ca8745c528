"""Page operations of a cache pool (byhip_cache_fork / _free / _grow / _compact / _copy) against the same steps
taken one after another on the host. Whole numbers and copied bytes: everything has to be equal."""
import numpy as np
import pytest

from bybylang_amd import _abi, synth

pytestmark = pytest.mark.gpu


class Pool:
    """The pool on the device and its host model."""

    def __init__(self, hip, slots, cols, pages, page, layers=2, Hk=2, D=8, seed=0):
        g = synth.rng(7400 + seed)
        self.hip, self.page, self.pages, self.cols, self.slots = hip, page, pages, cols, slots
        up = hip.DeviceBuffer.from_array
        self.kv = [[g.integers(0, 65536, (pages, Hk, page, D)).astype(np.uint16) for _ in range(2)] for _ in range(layers)]
        self.bufs = [[up(a) for a in pair] for pair in self.kv]
        self.table, self.refs, self.lens = np.full((slots, cols), -1, np.int32), np.zeros(pages, np.int32), np.zeros(slots, np.int32)
        self.status = np.zeros(4, np.int32)
        self.b = {k: up(getattr(self, k)) for k in ("table", "refs", "lens", "status")}
        caches = [hip.KvCache(k, v, hip.F16, pages, page, Hk, D) for k, v in self.bufs]
        self.dev = hip.KvPool(caches, self.b["refs"], self.b["table"], cols, self.b["lens"], slots, self.b["status"])

    def ints(self, v):
        return self.hip.DeviceBuffer.from_array(np.array(v if len(v) else [0], np.int32))

    def need(self, n):
        return -(-n // self.page)

    # the host model, entry after entry
    def fork(self, parents, rows):
        self.hip.cache_fork(self.dev, self.ints(parents), self.ints(rows), len(rows))
        self._assign(parents, rows)

    def free(self, rows):
        self.hip.cache_free(self.dev, self.ints(rows), len(rows))
        self._assign(None, rows)

    def _assign(self, parents, rows):
        table, lens = self.table.copy(), self.lens.copy()
        for i, r in enumerate(rows):
            a = parents[i] if parents is not None else None
            if not 0 <= r < self.slots or r in rows[:i] or (a is not None and (not 0 <= a < self.slots or a in rows)):
                self.status[1] += 1
                continue
            for p in self.table[r, :self.need(self.lens[r])]:
                self.refs[p] -= 1
            new = np.full(self.cols, -1, np.int32)
            if a is not None:
                n = self.need(self.lens[a])
                new[:n] = self.table[a, :n]
                for p in new[:n]:
                    self.refs[p] += 1
            table[r], lens[r] = new, 0 if a is None else self.lens[a]
        self.table, self.lens = table, lens

    def grow(self, rows, add):
        self.hip.cache_grow(self.dev, self.ints(rows), self.ints(add), len(rows))
        full, shrink = False, []
        for i, (r, n) in enumerate(zip(rows, add)):
            if not 0 <= r < self.slots or r in rows[:i]:
                self.status[1] += 1
                continue
            if n < 0:
                shrink.append((r, max(0, int(self.lens[r]) + n)))
                continue
            have, want = int(self.lens[r]), int(self.lens[r]) + n
            if n == 0:
                continue
            if want > self.cols * self.page:
                self.status[0] += 1
                continue
            part = have % self.page != 0
            copy = part and self.refs[self.table[r, have // self.page]] > 1
            cols = list(range(self.need(have) - copy, self.need(want)))
            free = np.flatnonzero(self.refs <= 0)[:len(cols)]
            if full or len(free) < len(cols):
                full = True
                self.status[0] += 1
                continue
            if copy:
                old = self.table[r, have // self.page]
                self.refs[old] -= 1
                self.status[2] += 1
                for pair in self.kv:
                    for a in pair:
                        a[free[0]] = a[old]
            for c, p in zip(cols, free):
                self.table[r, c] = p
                self.refs[p] = 1
            self.status[3] += len(cols)
            self.lens[r] = want
        for r, keep in shrink:
            for c in range(self.need(keep), self.need(self.lens[r])):
                self.refs[self.table[r, c]] -= 1
                self.table[r, c] = -1
            self.lens[r] = keep

    def compact(self, out=False):
        b_t, b_r = (self.hip.DeviceBuffer(self.table.nbytes), self.hip.DeviceBuffer(self.refs.nbytes)) if out else (None, None)
        self.hip.cache_compact(self.dev, b_t, b_r)
        live = int((self.refs > 0).sum())
        src = [p for p in range(live, self.pages) if self.refs[p] > 0]
        dst = [p for p in range(live) if self.refs[p] <= 0]
        table, refs = self.table.copy(), self.refs.copy()
        for s, d in zip(src, dst):
            table[self.table == s] = d
            refs[d], refs[s] = refs[s], 0
            for pair in self.kv:
                for a in pair:
                    a[d] = a[s]
        self.status[2] += len(src)
        if out:
            assert np.array_equal(b_t.read(np.int32).reshape(table.shape), table)
            assert np.array_equal(b_r.read(np.int32), refs)
            # adopt them, as a caller that swaps its buffers does
            self.b["table"].upload(table)
            self.b["refs"].upload(refs)
        self.table, self.refs = table, refs

    def check(self):
        for k in ("lens", "table", "refs", "status"):
            got = self.b[k].read(np.int32).reshape(getattr(self, k).shape)
            assert np.array_equal(got, getattr(self, k)), (k, got, getattr(self, k))
        for pair, bufs in zip(self.kv, self.bufs):
            for a, b in zip(pair, bufs):
                assert np.array_equal(b.read(np.uint16).reshape(a.shape), a)


def test_grow_fork_free(hip):
    p = Pool(hip, 8, 10, 40, 4)
    p.grow([0, 1, 2], [9, 4, 1])
    p.check()
    p.fork([0, 0, 1], [3, 4, 5])         # shared pages; slot 0's third page is partly filled
    p.check()
    p.grow([3, 0, 4, 5], [1, 1, 1, 1])   # two of its three holders copy it, the last keeps it
    p.check()
    assert p.status[2] == 2
    p.fork([2, 2], [3, 0])               # what the slots held is released
    p.free([1, 6])
    p.check()
    p.grow([5, 4], [-2, -100])           # the end is dropped
    p.check()
    p.free([0, 2, 3, 4, 5])
    p.check()
    assert not p.refs.any()


def test_lowest_pages_first_and_refusals_when_full(hip):
    p = Pool(hip, 5, 6, 7, 2)
    p.grow([0, 1, 2], [4, 4, 4])
    p.free([1])
    p.check()
    p.grow([3, 1, 4], [1, 9, 1])         # three pages are free: slot 3 fits, slot 1 does not, nor any after it
    p.check()
    assert p.status[0] == 2
    p.grow([3], [13])                    # more than the table's columns
    p.grow([0, 3], [0, 0])
    p.check()


def test_invalid_entries_change_nothing_else(hip):
    p = Pool(hip, 4, 4, 9, 2)
    p.grow([0, 9, 1, 0, -1], [3, 1, 2, 5, 1])
    p.check()
    p.fork([0, 7, 2, 0, 1], [2, 3, 3, 2, 1])  # parent out of range, parent among rows, twice, itself
    p.check()
    p.free([5, 1, 1, -3])
    p.check()
    p.grow([], [])
    p.fork([], [])
    p.check()


@pytest.mark.parametrize("seed", range(6))
def test_random_programs(hip, seed):
    g = synth.rng(7500 + seed)
    page = [1, 2, 4, 5, 16, 3][seed]
    slots, cols = int(g.integers(4, 90)), int(g.integers(4, 30))
    p = Pool(hip, slots, cols, int(g.integers(slots * 2, slots * cols)), page, layers=1 + seed % 3, Hk=1 + seed % 2, D=[8, 3, 16, 1, 8, 7][seed], seed=seed)
    for step in range(14):
        n = int(g.integers(1, slots))
        rows = g.permutation(slots)[:n].tolist()
        what = step % 4
        if what == 0:
            p.grow(rows, g.integers(-2 * page, 4 * page, n).tolist())
        elif what == 1:
            p.fork(g.integers(0, slots, n // 3 + 1).tolist(), rows[:n // 3 + 1])
        elif what == 2:
            p.grow(rows, g.integers(0, 2 * page + 1, n).tolist())
        else:
            p.free(rows[:n // 3])
            p.compact(out=step % 8 == 3)
        p.check()


def test_many_slots_and_pages(hip):
    p = Pool(hip, 1024, 4, 20000, 2, layers=1, Hk=1, D=2, seed=9)
    g = synth.rng(7600)
    p.refs[:] = (g.random(20000) < 0.8).astype(np.int32) * 3  # held by nobody here
    p.b["refs"].upload(p.refs)
    p.grow(list(range(1024)), g.integers(0, 8, 1024).tolist())
    p.check()
    p.compact()
    p.check()


@pytest.mark.parametrize("live", [0.0, 0.5, 1.0])
def test_compact_extremes(hip, live):
    p = Pool(hip, 3, 8, 24, 4, seed=11)
    if live:
        p.grow([0, 1, 2], [32, 32, 32] if live == 1.0 else [16, 13, 20])
    if live == 0.5:
        p.free([0])
    p.compact()
    p.check()


def test_page_copies_many_layers(hip):
    """More layers than one launch takes, pages of an odd size."""
    p = Pool(hip, 1, 1, 6, 3, layers=67, Hk=1, D=5, seed=12)
    src, dst = [0, 5, -1, 2, 9, 3], [1, 4, 2, 6, 3, 3]  # pairs outside the pool, and a page onto itself
    p.hip.cache_copy(p.dev, p.ints(src), p.ints(dst), 6)
    for pair in p.kv:
        for a in pair:
            a[1], a[4] = a[0], a[5]
    p.check()


def test_argument_refusals(hip):
    p = Pool(hip, 4, 4, 9, 2)
    E = _abi.HipBackendError
    one = p.ints([0])
    small = p.ints([0])
    bad = lambda **kw: hip.KvPool(**{**dict(caches=[hip.KvCache(*p.bufs[0], hip.F16, 9, 2, 2, 8)], refs=p.b["refs"], table=p.b["table"], table_stride=4,  # noqa: E731
                                            lens=p.b["lens"], slots=4, status=p.b["status"]), **kw})
    with pytest.raises(E, match="1025 slots"):
        hip.cache_grow(p.dev, one, one, 1025)
    with pytest.raises(E, match="-1 slots"):
        hip.cache_free(p.dev, one, -1)
    with pytest.raises(E, match="-1 page copies"):
        hip.cache_copy(p.dev, one, one, -1)
    with pytest.raises(E, match="slots needs"):
        hip.cache_free(p.dev, small, 2)
    with pytest.raises(E, match="parents needs"):
        hip.cache_fork(p.dev, small, p.ints([0, 1]), 2)
    with pytest.raises(E, match="token counts needs"):
        hip.cache_grow(p.dev, p.ints([0, 1]), small, 2)
    for match, kw in [("without caches", {"caches": []}), ("0 slots", {"slots": 0}), ("page table needs", {"slots": 99}), ("reference counts needs", {"refs": small}),
                      ("lengths needs", {"lens": small}), ("pool status needs", {"status": small}),
                      ("differs from the first", {"caches": [hip.KvCache(*p.bufs[0], hip.F16, 9, 2, 2, 8), hip.KvCache(*p.bufs[1], hip.F16, 9, 2, 1, 16)]}),
                      ("cache keys needs", {"caches": [hip.KvCache(*p.bufs[0], hip.F16, 90, 2, 2, 8)], "refs": hip.DeviceBuffer(400)})]:
        with pytest.raises(E, match=match):
            hip.cache_grow(bad(**kw), one, one, 1)
    with pytest.raises(E, match="moved page table needs"):
        hip.cache_compact(p.dev, small, None)
    _abi.load().byhip_fault_inject(1)
    with pytest.raises(E, match="injected fault"):
        hip.cache_compact(p.dev)
    p.check()
