"""PagedDecoder's steps, eager and replayed, against the block in 64 bits over what the device's cache holds, and the cache
against the keys and values that belong there: rows, positions and lengths that are one off show (tests/test_decoder_ref.py)."""
import numpy as np
import pytest

from bybylang_amd import _abi, synth
from decoder_ref import cached, keys_and_values, rows_of
from test_paged_decoder_gpu import DIM, HEADS, KV, PAGE, SLOTS, WIDTH, gb, make, matrices, split  # noqa: F401

pytestmark = pytest.mark.gpu


class Watched:
    """A decoder of one block, the rows that its slots were given, and the checks after each step."""

    def __init__(self, gb, pages=80):  # noqa: F811
        self.gb = gb
        self.d, ws, self.norms = make(gb, pages=pages)
        self.w = [matrices(gb, m) for m in ws[0]]
        self.seqs = [np.zeros((0, WIDTH), np.float32) for _ in range(SLOTS)]

    def cache(self, slot):
        """The keys and values of a slot's tokens, [L, KV, DIM]."""
        d, n, L = self.d, self.d.caches[0].value, len(self.seqs[slot])
        table = self.gb.sessionRead(self.gb.gbHip, d.table, SLOTS * d.stride).view(np.int32).reshape(SLOTS, -1)[slot]
        at = np.arange(L)
        shape = (n.pages, KV, PAGE, DIM)
        return [self.gb.sessionRead(self.gb.gbHip, b, int(np.prod(shape)) // 2).view(np.float16).reshape(shape)[table[at // PAGE], :, at % PAGE].astype(np.float64)
                for b in d.caches[0].keep[:2]]

    def check(self, x, counts, got, what):
        for i, part in enumerate(split(x, counts)):
            self.seqs[i] = np.concatenate([self.seqs[i], part])
        assert self.d.lengths().tolist() == [len(s) for s in self.seqs]
        for i, rows in enumerate(split(got, counts)):
            if not len(self.seqs[i]):
                continue
            k, v = self.cache(i)
            wk, ek, wv, ev = keys_and_values(self.w, self.norms, self.seqs[i], KV)
            assert cached(k, wk, ek) <= 1 and cached(v, wv, ev) <= 1, f"{what}: the cache of slot {i}: {cached(k, wk, ek):.3g}, {cached(v, wv, ev):.3g} of the bound"
            if counts[i]:
                y, bound = rows_of(self.w, self.norms, self.seqs[i], k, v, counts[i], HEADS)
                worst = np.max(np.abs(rows - y) / bound)
                assert worst <= 1, f"{what}: slot {i}: {worst:.3g} of the bound"

    def run(self, x, counts, what):
        self.check(x, counts, self.d.forward(x, counts), what)


def rows(rng, n):
    return rng.standard_normal((n, WIDTH)).astype(np.float32)


def test_prompts_steps_forks_and_compaction(gb):  # noqa: F811
    t, rng = Watched(gb), synth.rng(41)
    t.run(rows(rng, 126), [5, 0, 33, 1, 70, 17], "prompts")
    t.run(rows(rng, 63), [1, 40, 1, 20, 1, 0], "chunks beside steps")
    for i in range(4):
        t.run(rows(rng, SLOTS), [1] * SLOTS, f"step {i}")
    t.d.free([1, 3])
    t.d.fork([4, 4], [1, 3])
    t.seqs[1], t.seqs[3] = t.seqs[4], t.seqs[4]
    for i in range(3):
        t.run(rows(rng, SLOTS), [1] * SLOTS, f"forked step {i}")
    t.d.free([0, 4])
    t.seqs[0] = t.seqs[4] = t.seqs[0][:0]
    t.d.compact()
    t.run(rows(rng, 4), [0, 1, 1, 1, 0, 1], "steps after compaction")
    t.run(rows(rng, 77), [64, 1, 0, 2, 9, 1], "prompts in freed slots")
    assert t.d.refused() == 0


@pytest.mark.parametrize("direct", [False, True], ids=["graph", "direct"])
def test_replayed_steps(gb, direct):  # noqa: F811
    _abi.check(_abi.load().byhip_session_set_direct_replay(int(direct)))
    t, rng = Watched(gb), synth.rng(42)
    t.run(rows(rng, 126), [5, 0, 33, 1, 70, 17], "prompts")
    x = rows(rng, SLOTS)
    t.d.set_rows([1] * SLOTS)
    t.d.set_input(x)
    step = t.d.record()
    t.check(x, [1] * SLOTS, t.d.output(), "the recorded step")
    for i in range(20):
        x = rows(rng, SLOTS)
        t.d.set_input(x)
        assert gb.sessionReplay(gb.gbHip, step, 1), gb.sessionGetLastError(gb.gbHip)
        t.check(x, [1] * SLOTS, t.d.output(), f"replay {i}")
    gb.sessionFreeRecording(gb.gbHip, step)
