"""A batch whose last sequences have rows past the call's `rows`: the sequence that the limit cuts is left out whole, by
byhip_rope_append and by every kernel of byhip_paged_attention."""
import numpy as np
import pytest

from bybylang_amd import _abi, synth
from paged_ref import from_bits, paged, to_bits
from test_attn_gpu import Case

pytestmark = pytest.mark.gpu
F32, F16, BF16 = _abi.F32, _abi.F16, _abi.BF16


@pytest.mark.parametrize("D", [64, 20, 260])  # attn_rows and attn_chunk; attn_general
@pytest.mark.parametrize("new", [[1, 2, 3], [1, 60, 40]])
def test_attention_leaves_out_a_sequence_that_is_cut(hip, D, new):
    c = Case(hip, [90, 70, 80], new, 4, 2, D, 16, F16, F32, F32)
    up = hip.DeviceBuffer.from_array
    bufs = [up(a) for a in (c.q, c.kv[0], c.kv[1], c.table, c.starts, np.array(c.lens, np.int32))]
    q, k, v, t, s, n = bufs
    out = up(np.full((c.T, c.W), 77.0, np.float32))
    rows = int(c.starts[2]) + 1  # the first row of the last sequence, but not the others
    hip.paged_attention(q, c.W, F32, 4, hip.Attn(c.scale), hip.KvCache(k, v, F16, c.pages, 16, 2, D),
                        hip.KvBatch(t, c.table.shape[1], s, n, 3, rows), out, c.W, F32)
    got = out.read(np.float32, c.T * c.W).reshape(c.T, 4, D)
    assert np.all(got[rows - 1:] == 77.0)
    c.new = new[:2] + [0]
    c.check(got.astype(np.float64))


@pytest.mark.parametrize("D,pad", [(64, 0), (20, 1)])
def test_rope_leaves_out_a_sequence_that_is_cut(hip, D, pad):
    g = synth.rng(8100 + D)
    H, Hk, page, lens, new = 3, 1, 4, [9, 6, 8], [2, 3, 4]
    pages = sum(-(-n // page) for n in lens) + 2
    table, W = paged(g, lens, page, pages), (H + 2 * Hk) * D + pad
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    x = to_bits(g.standard_normal((sum(new), W)), F16)
    kv = [to_bits(g.standard_normal((pages, Hk, page, D)), F16) for _ in range(2)]
    steps, _ = hip.rope_steps(D)
    up = hip.DeviceBuffer.from_array
    bx, bk, bv, bt, bs, bl, bsteps = up(x), up(kv[0]), up(kv[1]), up(table), up(starts), up(np.array(lens, np.int32)), up(steps)

    class At:
        def __init__(self, off):
            self.ptr = bx.ptr + 2 * off

    def run(rows, batch):
        bk.upload(kv[0])
        bv.upload(kv[1])
        out = up(np.full((sum(new), H * D), 5, np.float16))
        hip.rope_append(At(0), W, At(H * D), W, At((H + Hk) * D), W, F16, H, hip.Rope(_abi.ROPE_HALVES, D, bsteps), hip.KvCache(bk, bv, F16, pages, page, Hk, D),
                        hip.KvBatch(bt, table.shape[1], bs, bl, batch, rows), out, H * D, F16)
        return out.read(np.float16), bk.read(np.float16), bv.read(np.float16)
    for a, b in zip(run(6, 3), run(5, 2)):  # one row of the third sequence; without the third sequence
        assert np.array_equal(from_bits(a, F16), from_bits(b, F16))
