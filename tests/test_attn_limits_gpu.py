"""byhip_paged_attention at the ends of its numbers: empty and tiny queries, infinite keys and values that
are seen, windows near 2^31."""
import numpy as np
import pytest

from bybylang_amd import _abi
from paged_ref import attention, close, from_bits, to_bits
from test_attn_gpu import Case

pytestmark = pytest.mark.gpu
F32, F16, BF16 = _abi.F32, _abi.F16, _abi.BF16


@pytest.mark.parametrize("new", [1, 20, 200])
@pytest.mark.parametrize("ct", [F16, BF16])
@pytest.mark.parametrize("scale", [None, 2.0**-11, 1e-20, 1e-38])
@pytest.mark.parametrize("value", [0.0, 1e-42, 1e-38, 1e-30])
def test_empty_and_tiny_queries(hip, new, ct, scale, value):
    """Rows of padding have queries of zeros: they weigh the keys that they see alike, and no others."""
    c = Case(hip, [230], [new], 4, 2, 128, 32, ct, F32, F32, seed=20, scale=scale)
    c.q[::2] = np.float32(value) * np.sign(c.q[::2])
    c.check()


@pytest.mark.parametrize("new", [1, 20, 200])
@pytest.mark.parametrize("D", [20, 64, 128, 256])
@pytest.mark.parametrize("ct,qt,ot", [(F16, F32, F32), (BF16, F32, F32), (F16, F16, F32), (F16, F16, F16), (BF16, BF16, BF16)])
def test_keys_of_minus_infinity_have_no_weight(hip, new, D, ct, qt, ot):
    c = Case(hip, [260], [new], 4, 2, D, 16, ct, qt, ot, seed=21)
    rows = from_bits(c.q, qt)
    rows[:, 5::D] = np.abs(rows[:, 5::D]) + 2.0**-9
    rows[:, 9::D] = -2.0**-45 if qt == F32 else -2.0**-9  # 2^-45: below half of fp16's least value in its row's scale
    c.q = to_bits(rows, qt)
    inf = to_bits(np.array([np.inf, -np.inf]), ct)
    low = np.zeros(260, bool)
    for j, d, s in ((3, 5, 1), (40, 5, 1), (41, 9, 0), (59, 5, 1)):
        c.kv[0][c.table[0, j // 16], :, j % 16, d] = inf[s]
        low[j] = True
    got = c.run()
    q = from_bits(c.q, qt).reshape(-1, 4, D)
    k, v, there = c.sequence(0)
    k = np.where(np.isfinite(k), k, 0)
    out, mean, size, flat = attention(q, k, v, float(np.float32(c.scale)), 0, 0, None, 0, ~low)
    slack = (2 * np.sqrt(D) * 2.0**-24 * size + 4e-6 + np.sqrt(260) * 2.0**-22) * (mean + np.abs(out))
    if F32 not in (qt, ot):
        slack = slack + {F16: 2.0**-11, BF16: 2.0**-8}[ct] * mean + (2.0**-25 * flat if ct == F16 else 0)
    close(got, out, ot, slack)


def test_rows_whose_scores_are_all_minus_infinity(hip):
    for new in (1, 20, 200):
        for ct in (F16, BF16):
            c = Case(hip, [230], [new], 4, 2, 64, 16, ct, F32, F32, seed=22)
            c.q[:, 7::64] = np.abs(c.q[:, 7::64]) + 1
            c.kv[0][..., 7] = to_bits(np.array([-np.inf]), ct)[0]
            assert np.all(c.run() == 0)


@pytest.mark.parametrize("new", [1, 20, 200])
@pytest.mark.parametrize("D", [20, 64, 128, 256])
@pytest.mark.parametrize("ct,qt", [(F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)])
def test_infinite_values_show_however_small_their_weight(hip, new, D, ct, qt):
    """A key that is seen has a weight above 0: an infinite value of it is the sum."""
    c = Case(hip, [300], [new], 2, 1, D, 16, ct, qt, qt, seed=23, scale=1.0)
    c.q = to_bits(np.abs(from_bits(c.q, qt)) + 0.5, qt)
    top = from_bits(c.q, qt).reshape(-1, 2, D).sum(-1)
    at = lambda j: (c.table[0, j // 16], slice(None), j % 16)  # noqa: E731
    c.kv[0][at(37)] = to_bits(np.full((1, D), -240.0 / top.min()), ct)  # a score at least 120 below the others'
    c.kv[0][at(38)] = to_bits(np.full((1, D), 120.0 / top.min()), ct)
    c.kv[1][at(37)] = to_bits(np.where(np.arange(D) == 7, np.inf, np.where(np.arange(D) == 8, -np.inf, 1.0))[None], ct)
    got = c.run()
    assert np.all(got[..., 7] == np.inf) and np.all(got[..., 8] == -np.inf)
    assert np.all(np.isfinite(np.delete(got, [7, 8], -1)))


@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 4, 2**31 - 40])
@pytest.mark.parametrize("prefix", [None, [30]])
@pytest.mark.parametrize("beside", [0, 199])
def test_windows_near_the_largest_number(hip, window, prefix, beside):
    """More rows than tokens, so that the first rows' positions lie below 0: no window of this size hides a key."""
    c = Case(hip, [130], [130], 2, 1, 64, 16, F16, F32, F32, seed=24, window=window, prefix=None if prefix is None else prefix + [0] * beside)
    c.lens, c.new = [100] + [0] * beside, c.new + [0] * beside
    c.table = np.concatenate([c.table, np.full((beside, c.table.shape[1]), -1, np.int32)])
    c.starts = np.concatenate([c.starts, np.full(beside, c.starts[-1], np.int32)])
    c.check()
