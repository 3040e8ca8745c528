"""The operators of a paged cache run together (bybylang_amd/paged_decoder.py): ragged prompts, decode steps,
forks, ends and compaction against the blocks in 64 bits; recorded steps, replayed, against the same steps
run eagerly; and no device memory allocated by any of them.
"""
import numpy as np
import pytest

from bybylang_amd import _abi, synth

pytestmark = pytest.mark.gpu

WIDTH, HEADS, KV, DIM, SLOTS, MAX_LEN, MAX_ROWS, PAGE = 256, 8, 2, 64, 6, 160, 256, 16
EPS = 1e-5


@pytest.fixture
def gb(hip):
    from bybylang_amd import gpubackend as g
    yield g
    g.sessionRecoverQueue(g.gbHip)
    _abi.check(_abi.load().byhip_session_set_direct_replay(0))


def matrices(gb, w):
    """The weights a resident matrix multiplies by, [K][N]: its product with the unit matrix."""
    x = gb.sessionUpload(gb.gbHip, np.eye(w.k, dtype=np.float32).reshape(-1))
    y = gb.sessionAllocScratch(gb.gbHip, w.k * w.n)
    assert gb.sessionMatmulQ4(gb.gbHip, x, w, y, w.k)
    return gb.sessionRead(gb.gbHip, y, w.k * w.n).reshape(w.k, w.n).astype(np.float64)


def make(gb, layers=1, pages=80, seed=5):
    from bybylang_amd import paged_decoder as p
    rng = synth.rng(seed)
    ws = [(p.random_weights(rng, WIDTH, HEADS * DIM), p.random_weights(rng, WIDTH, KV * DIM),
           p.random_weights(rng, WIDTH, KV * DIM), p.random_weights(rng, HEADS * DIM, WIDTH)) for _ in range(layers)]
    norms = [rng.uniform(0.5, 1.5, WIDTH).astype(np.float32) for _ in range(layers + 1)]
    return p.PagedDecoder(ws, norms, WIDTH, HEADS, KV, DIM, SLOTS, MAX_LEN, MAX_ROWS, pages, PAGE), ws, norms


def rotated(x, pos):
    """Rotary positions over halves, base 10000."""
    i = np.arange(DIM // 2)
    angle = pos[:, None] * 10000.0 ** (-2.0 * i / DIM)
    c, s = np.cos(angle)[:, None, :], np.sin(angle)[:, None, :]
    a, b = x[..., : DIM // 2], x[..., DIM // 2:]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def block(w, norms, x):
    """One layer over a sequence's rows x in 64 bits, and what fp32 products with a cache of fp16 may be off by: a
    key or value is off by 2^-11 of itself (rounding; a bit more for the fp32 arithmetic before it), a score by the sum
    of those, a weight by the score's factor twice (it and the sum it is divided by), and each product by 2^-18 of its terms."""
    wq, wk, wv, wo = w
    x = x.astype(np.float64)
    n, unit, dot = len(x), 2.0**-11 + 2.0**-14, 2.0**-18
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * norms[0]
    pos = np.arange(n)
    q, k = rotated((y @ wq).reshape(n, HEADS, DIM), pos), rotated((y @ wk).reshape(n, KV, DIM), pos)
    v = (y @ wv).reshape(n, KV, DIM)
    a, ea = np.zeros((n, HEADS, DIM)), np.zeros((n, HEADS, DIM))
    fuzz = dot * np.abs(y).sum(-1).max() * max(np.abs(wq).max(), np.abs(wk).max(), np.abs(wv).max())  # of q, k and v
    for h in range(HEADS):
        kh, vh = k[:, h // (HEADS // KV)], v[:, h // (HEADS // KV)]
        s = q[:, h] @ kh.T * DIM**-0.5
        s[pos[None, :] > pos[:, None]] = -np.inf
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        a[:, h] = p @ vh
        off = (np.abs(q[:, h]) @ np.abs(kh).T * unit + fuzz * (np.abs(q[:, h]).sum(-1)[:, None] + np.abs(kh).sum(-1)[None, :])) * DIM**-0.5
        off = np.where(pos[None, :] <= pos[:, None], off, 0).max(-1)
        ea[:, h] = unit * (p @ np.abs(vh)) + fuzz + np.expm1(2 * off)[:, None] * (p @ np.abs(vh))
    a, ea = a.reshape(n, -1), ea.reshape(n, -1)
    h = x + a @ wo
    eh = ea @ np.abs(wo) + dot * (np.abs(a) @ np.abs(wo)) + 2.0**-22 * np.abs(h)
    rms = np.sqrt((h * h).mean(-1, keepdims=True) + EPS)
    y = h / rms * norms[1]
    ey = (eh * np.abs(norms[1]) + np.abs(y) * np.sqrt((eh * eh).mean(-1, keepdims=True))) / rms + 2.0**-20 * np.abs(y)
    return y, 1.1 * ey


def agree(got, want, what):
    y, bound = want
    off = np.abs(got - y)
    assert (off <= bound).all(), f"{what}: worst {np.max(off / bound):.3g} of the bound"


def split(rows, counts):
    return np.split(rows, np.cumsum(counts)[:-1])


def test_prompts_steps_forks_and_compaction_against_64_bits(gb):
    d, ws, norms = make(gb)
    w = [matrices(gb, m) for m in ws[0]]
    rng = synth.rng(6)
    seqs = [np.zeros((0, WIDTH), np.float32) for _ in range(SLOTS)]

    def run(counts, what):
        x = rng.standard_normal((sum(counts), WIDTH)).astype(np.float32)
        got = split(d.forward(x, counts), counts)
        for i, part in enumerate(split(x, counts)):
            seqs[i] = np.concatenate([seqs[i], part])
            if counts[i]:
                y, bound = block(w, norms, seqs[i])
                agree(got[i], (y[-counts[i]:], bound[-counts[i]:]), f"{what}, slot {i}")
        assert d.lengths().tolist() == [len(s) for s in seqs]

    run([5, 0, 33, 1, 70, 17], "prompts")
    run([1, 40, 1, 20, 1, 0], "chunks beside steps")
    run([1] * SLOTS, "steps")
    d.free([1, 3])
    d.fork([4, 4], [1, 3])  # two beams of slot 4 share its pages
    seqs[1], seqs[3] = seqs[4], seqs[4]
    run([1] * SLOTS, "forked steps")
    d.free([0, 4])
    seqs[0] = seqs[4] = seqs[0][:0]
    d.compact()
    run([0, 1, 1, 1, 0, 1], "steps after compaction")
    run([64, 1, 0, 2, 9, 1], "prompts in freed slots")
    assert d.refused() == 0


@pytest.mark.parametrize("direct", [False, True], ids=["graph", "direct"])
def test_replayed_steps_equal_eager_ones(gb, direct):
    _abi.check(_abi.load().byhip_session_set_direct_replay(int(direct)))
    eager, ws, _ = make(gb, layers=2)
    kept, _, _ = make(gb, layers=2)
    rng = synth.rng(7)
    counts = [5, 0, 33, 1, 70, 17]
    x = rng.standard_normal((sum(counts), WIDTH))
    assert np.array_equal(eager.forward(x, counts), kept.forward(x, counts))
    xs = rng.standard_normal((6, SLOTS, WIDTH))
    want = [eager.forward(xs[0], [1] * SLOTS)]
    assert np.array_equal(kept.forward(xs[0], [1] * SLOTS), want[0])
    before = kept.lengths()
    step = kept.record()
    ran = int((kept.lengths() - before).max())  # whether recording a step is also a step
    at = 1
    if ran:
        want.append(eager.forward(xs[0], [1] * SLOTS))
        assert np.array_equal(kept.output(), want[-1])
    for at in range(1, 6):
        kept.set_input(xs[at])
        assert gb.sessionReplay(gb.gbHip, step, 1), gb.sessionGetLastError(gb.gbHip)
        got = kept.output()
        assert np.array_equal(got, eager.forward(xs[at], [1] * SLOTS)), f"step {at}"  # eager work between the replays
    assert kept.lengths().tolist() == eager.lengths().tolist()
    gb.sessionFreeRecording(gb.gbHip, step)


def test_steps_allocate_nothing(gb):
    d, _, _ = make(gb, layers=2)
    rng = synth.rng(8)
    counts = [5, 0, 33, 1, 70, 17]
    lib = _abi.load()

    def all_of_it():
        d.forward(rng.standard_normal((sum(counts), WIDTH)), counts)
        d.forward(rng.standard_normal((SLOTS, WIDTH)), [1] * SLOTS)
        d.free([1])
        d.fork([4], [1])
        d.free(range(SLOTS))
        d.compact()

    all_of_it()  # the matmuls' scratch, once
    before = lib.byhip_debug_alloc_count()
    all_of_it()
    assert lib.byhip_debug_alloc_count() == before


def test_session_procs_say_what_they_do_not_take(gb):
    from bybylang_amd import device as dev
    d, _, _ = make(gb)
    d.set_rows([1] * SLOTS)
    odd = dev.KvCache(d.caches[0].keep[0], d.caches[0].keep[1], _abi.F32, 80, PAGE, KV, DIM)
    assert not gb.sessionPagedAttention(gb.gbHip, d.q, HEADS, d.attn, odd, d.batch, d.a)
    with pytest.raises(_abi.HipBackendError):
        gb.sessionPagedAttention(gb.gbHip, d.q, 7, d.attn, d.caches[0], d.batch, d.a)  # 7 heads over 2 key heads
    with pytest.raises(ValueError):
        gb.sessionNormBlock(gb.gbCpu, d.x, 1, WIDTH, None, None, None, 1.0, d.h, d.norms[0], d.y)
