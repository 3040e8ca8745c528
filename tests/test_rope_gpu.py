"""byhip_rope_append against the rotation in 64 bits, through device.rope_append.

Bound on a rotated value (a, b): the angle's fraction keeps 24 bits of at most pi / 4 and the sine's and cosine's Taylor
sums are off by at most 3e-8 and their own roundings, together under 2.5e-7; three more roundings of products
no larger than m (|a| + |b|) add 1.8e-7. So 5e-7 m (|a| + |b|) and the output's rounding. Values are copied bit for bit.
"""
import numpy as np
import pytest

from bybylang_amd import _abi, synth
from paged_ref import close, from_bits, paged, rope, rounded, to_bits

pytestmark = pytest.mark.gpu
F32, F16, BF16 = _abi.F32, _abi.F16, _abi.BF16
HALVES, PAIRS = _abi.ROPE_HALVES, _abi.ROPE_PAIRS


def case(hip, lens, new, H, Hk, D, page, rot, layout, xt, ct, qt, pad=0, mag=1.0, seed=0, cols=0):
    g = synth.rng(4100 + seed)
    T, W = sum(new), (H + 2 * Hk) * D + pad
    pages = sum(-(-n // page) for n in lens) + 3
    table = paged(g, lens, page, pages, cols)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    x = to_bits(g.standard_normal((T, W)), xt)
    kv = [to_bits(g.standard_normal((pages, Hk, page, D)), ct) for _ in range(2)]
    steps, _ = hip.rope_steps(rot)
    up = hip.DeviceBuffer.from_array
    bx, bk, bv, bt, bs, bl = up(x), up(kv[0]), up(kv[1]), up(table), up(starts), up(np.array(lens, np.int32))
    bsteps = up(steps if rot else np.zeros(1, np.uint64))
    size = 4 if xt == F32 else 2

    class At:
        def __init__(self, off):
            self.ptr = bx.ptr + off * size
    cache = hip.KvCache(bk, bv, ct, pages, page, Hk, D)
    batch = hip.KvBatch(bt, table.shape[1], bs, bl, len(lens), T)
    out = hip.DeviceBuffer(max(1, T * H * D * (4 if qt == F32 else 2)))
    hip.rope_append(At(0), W, At(H * D), W, At((H + Hk) * D), W, xt, H, hip.Rope(layout, rot, bsteps, mag), cache, batch, out, H * D, qt)
    np_of = {F32: np.float32, F16: np.float16, BF16: np.uint16}
    got_q = from_bits(out.read(np_of[qt], T * H * D), qt).reshape(T, H, D)
    got = [b.read(np_of[ct], a.size).reshape(a.shape) for b, a in zip((bk, bv), kv)]
    rows = from_bits(x, xt)[:, :(H + 2 * Hk) * D].reshape(T, H + 2 * Hk, D)
    want_k, bound_k = from_bits(kv[0], ct), np.zeros(kv[0].shape)
    want_v = kv[1].copy()
    for b, (L, n) in enumerate(zip(lens, new)):
        t = slice(starts[b], starts[b] + n)
        pos = np.arange(L - n, L)
        y = rope(rows[t], pos, steps, rot, layout, mag) if n else rows[t]
        size_of = np.abs(rows[t]).copy()
        a, c = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == HALVES else (slice(0, rot, 2), slice(1, rot, 2))
        both = (size_of[..., a] + size_of[..., c]) * mag
        size_of[..., a], size_of[..., c] = both, both
        size_of[..., rot:] = 0
        close(got_q[t], y[:, :H], qt, 5e-7 * size_of[:, :H], "q")
        pg, sl = table[b, pos // page], pos % page
        want_k[pg, :, sl] = y[:, H:H + Hk]
        bound_k[pg, :, sl] = 5e-7 * size_of[:, H:H + Hk]
        want_v[pg, :, sl] = to_bits(rows[t][:, H + Hk:], ct)
    untouched = bound_k == 0
    close(from_bits(got[0], ct), want_k, ct, bound_k, "k")
    assert np.array_equal(from_bits(got[0], ct)[untouched & (want_k == from_bits(kv[0], ct))], want_k[untouched & (want_k == from_bits(kv[0], ct))])
    assert np.array_equal(got[1], want_v), "v"


@pytest.mark.parametrize("xt,ct,qt", [(F32, F16, F32), (F32, BF16, BF16), (F16, F16, F16), (BF16, BF16, F32)])
@pytest.mark.parametrize("layout", [HALVES, PAIRS])
def test_types_and_layouts(hip, xt, ct, qt, layout):
    case(hip, [1, 40, 131, 7], [1, 3, 20, 0], 8, 2, 128, 16, 128, layout, xt, ct, qt, seed=xt * 9 + qt)


@pytest.mark.parametrize("D,rot,pad", [(128, 64, 0), (80, 40, 0), (64, 64, 4), (64, 32, 3), (37, 20, 0), (96, 90, 1), (256, 256, 0), (8, 0, 0), (1, 0, 0), (2, 2, 0), (600, 520, 0)])
@pytest.mark.parametrize("layout", [HALVES, PAIRS])
def test_head_dims_parts_and_strides(hip, D, rot, pad, layout):
    case(hip, [33, 5], [9, 5], 3, 1, D, 5, rot, layout, F32, F16, F32, pad=pad, mag=1.2, seed=D)


@pytest.mark.parametrize("batch", [1, 63, 64, 65, 130, 4097])
def test_batches_and_empty_sequences(hip, batch):
    """Row searches over one, two and three levels; every third sequence brings nothing."""
    new = [0 if b % 3 == 1 else 1 + b % 2 for b in range(batch)]
    case(hip, [n + b % 5 for b, n in enumerate(new)], new, 2, 1, 16, 4, 16, HALVES, F16, F16, F16, seed=batch, cols=1)


def test_far_positions(hip):
    """Positions whose fp32 product with a frequency would be off by 0.1 rad and more."""
    g = synth.rng(4199)
    H, D, L = 2, 64, 2**31 - 5
    x = g.standard_normal((3, H * D)).astype(np.float32)
    steps, _ = hip.rope_steps(D)
    up = hip.DeviceBuffer.from_array
    batch = hip.KvBatch(up(np.zeros(1, np.int32)), 1, up(np.array([0, 3], np.int32)), up(np.array([L], np.int32)), 1, 3)
    out = hip.DeviceBuffer(x.nbytes)
    hip.rope_append(up(x), H * D, None, 0, None, 0, F32, H, hip.Rope(PAIRS, D, up(steps)), None, batch, out, H * D, F32, head_dim=D)
    rows = x.astype(np.float64).reshape(3, H, D)
    both = np.repeat(np.abs(rows[..., 0::2]) + np.abs(rows[..., 1::2]), 2, axis=-1)
    close(out.read(np.float32).reshape(3, H, D), rope(rows, np.arange(L - 3, L), steps, D, PAIRS, 1.0), F32, 5e-7 * both)


def test_in_place_and_unrotated(hip):
    g = synth.rng(4198)
    x = g.standard_normal((4, 64)).astype(np.float32)
    steps, _ = hip.rope_steps(32)
    up = hip.DeviceBuffer.from_array
    batch = hip.KvBatch(up(np.zeros(1, np.int32)), 1, up(np.array([0, 4], np.int32)), up(np.array([9], np.int32)), 1, 4)
    b = up(x)
    hip.rope_append(b, 64, None, 0, None, 0, F32, 2, hip.Rope(HALVES, 32, up(steps)), None, batch, b, 64, F32, head_dim=32)
    rows = x.astype(np.float64).reshape(4, 2, 32)
    both = np.tile(np.abs(rows[..., :16]) + np.abs(rows[..., 16:]), 2)
    close(b.read(np.float32).reshape(4, 2, 32), rope(rows, np.arange(5, 9), steps, 32, HALVES, 1.0), F32, 5e-7 * both)
    b = up(x)
    out = hip.DeviceBuffer(4 * 64 * 2)
    hip.rope_append(b, 64, None, 0, None, 0, F32, 2, None, None, batch, out, 64, F16, head_dim=32)
    assert np.array_equal(out.read(np.float16).reshape(4, 64), x.astype(np.float16))


def test_what_lies_outside_is_left_out(hip):
    """Pages outside the pool, positions outside the table or below 0: nothing is written for them."""
    g = synth.rng(4197)
    H = Hk = 1
    D, page, pages = 8, 4, 3
    up = hip.DeviceBuffer.from_array
    kv = np.full((pages, Hk, page, D), 7, np.float16)
    bk, bv = up(kv), up(kv)
    table = np.array([[1, 3], [-1, 2], [0, 0]], np.int32)  # page 3 and -1 do not exist
    lens, new = [6, 2, 30], [6, 2, 2]                      # sequence 2 ends past its table
    starts = np.array([0, 6, 8, 10], np.int32)
    x = g.standard_normal((10, 3 * D)).astype(np.float16)
    b = up(x)

    class At:
        def __init__(self, o):
            self.ptr = b.ptr + 2 * o
    out = up(np.full((10, D), 5, np.float16))
    batch = hip.KvBatch(up(table), 2, up(starts), up(np.array(lens, np.int32)), 3, 10)
    hip.rope_append(At(0), 3 * D, At(D), 3 * D, At(2 * D), 3 * D, F16, 1, None, hip.KvCache(bk, bv, F16, pages, page, 1, D), batch, out, D, F16)
    want = kv.copy()
    want[1, 0] = x[:4, D:2 * D]
    assert np.array_equal(bk.read(np.float16).reshape(kv.shape), want)
    assert np.array_equal(out.read(np.float16).reshape(10, D), x[:, :D])
    # more rows than tokens: the first has position -1
    out = up(np.full((3, D), 5, np.float16))
    batch = hip.KvBatch(up(table), 2, up(np.array([0, 3], np.int32)), up(np.array([2], np.int32)), 1, 3)
    hip.rope_append(At(0), 3 * D, None, 0, None, 0, F16, 1, None, None, batch, out, D, F16, head_dim=D)
    got = out.read(np.float16).reshape(3, D)
    assert np.all(got[0] == 5) and np.array_equal(got[1:], x[1:3, :D])


def test_refusals(hip):
    up = hip.DeviceBuffer.from_array
    z = up(np.zeros(4096, np.float32))
    small = up(np.zeros(4, np.float32))
    ints = up(np.zeros(64, np.int32))
    batch = hip.KvBatch(ints, 4, ints, ints, 2, 4)
    cache = hip.KvCache(z, z, F16, 2, 4, 1, 16)
    steps = up(np.zeros(8, np.uint64))

    def call(heads=2, rope=None, c=cache, bt=batch, q=z, qs=32, ks=16, xt=F32, out=z, os=32, ot=F16, hd=0):
        hip.rope_append(q, qs, z, ks, z, 16, xt, heads, rope, c, bt, out, os, ot, head_dim=hd)
    ok = up(np.zeros(1024, np.float32))
    call(out=ok)
    E, U = _abi.HipBackendError, _abi.HipUnsupported
    for err, match, kw in [
            (E, "0 heads", {"heads": 0}), (E, "stride 8 below", {"qs": 8}), (E, "stride 4 below", {"ks": 4}), (E, "dtype 3", {"xt": 3}),
            (E, "dtype 7", {"ot": 7}), (E, "needs .* bytes", {"q": small}), (E, "needs .* bytes", {"out": small}),
            (E, "rotary layout", {"rope": hip.Rope(5, 8, steps)}), (E, "18 of 16", {"rope": hip.Rope(0, 18, steps)}),
            (E, "3 of 16", {"rope": hip.Rope(0, 3, steps)}), (E, "needs .* bytes", {"rope": hip.Rope(0, 16, small)}),
            (U, "fp16 or bf16", {"c": hip.KvCache(z, z, F32, 2, 4, 1, 16)}), (E, "cache of 0 pages", {"c": hip.KvCache(z, z, F16, 0, 4, 1, 16)}),
            (E, "cache keys needs", {"c": hip.KvCache(small, z, F16, 2, 4, 1, 16)}), (E, "the cache's of 16", {"hd": 8}),
            (E, "page table needs", {"bt": hip.KvBatch(ints, 40, ints, ints, 2, 4)}), (E, "row starts needs", {"bt": hip.KvBatch(z, 1, small, z, 8, 4)}),
            (E, "-1 rows", {"bt": hip.KvBatch(ints, 4, ints, ints, 2, -1)}), (E, "in place", {"out": z})]:
        with pytest.raises(err, match=match):
            call(**{"out": ok, **kw})
    _abi.load().byhip_fault_inject(1)
    with pytest.raises(E, match="injected fault"):
        call(out=ok)
