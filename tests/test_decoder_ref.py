"""The oracle of the decoder's steps has bounds that mistakes do not fit into (no GPU): the mistakes are planted in the oracle."""
import numpy as np
import pytest

from bybylang_amd import synth
from decoder_ref import cached, keys_and_values, rows_of

WIDTH, HEADS, KV, DIM = 256, 8, 2, 64


def case(L, seed=3):
    """Weights as PagedDecoder's random ones, a sequence and its cache."""
    g = synth.rng(seed)

    def weights(K, N):
        return ((g.integers(0, 16, (K, N)) - 7.5) * np.repeat(g.uniform(0.5, 1.5, (K // 32, N)), 32, 0) * 0.2 / np.sqrt(K))
    w = [weights(WIDTH, HEADS * DIM), weights(WIDTH, KV * DIM), weights(WIDTH, KV * DIM), weights(HEADS * DIM, WIDTH)]
    norms = [g.uniform(0.5, 1.5, WIDTH).astype(np.float32) for _ in range(2)]
    x = g.standard_normal((L, WIDTH)).astype(np.float32)
    k, _, v, _ = keys_and_values(w, norms, x, KV)
    return w, norms, x, k.astype(np.float16).astype(np.float64), v.astype(np.float16).astype(np.float64)


@pytest.mark.parametrize("L", [2, 17, 40, 100, 160])
@pytest.mark.parametrize("n", [1, 16])
@pytest.mark.parametrize("mistake", [dict(turn=1), dict(turn=-1), dict(share=0.5), dict(share=0.9), dict(drop=1)], ids=str)
def test_mistakes_in_rows_are_past_the_bound(L, n, mistake):
    w, norms, x, k, v = case(L)
    n = min(n, L - 1)  # a row 0 with its only key dropped has no attention
    y, bound = rows_of(w, norms, x, k, v, n, HEADS)
    wrong, _ = rows_of(w, norms, x, k, v, n, HEADS, **mistake)
    assert np.all(np.max(np.abs(wrong - y) / bound, axis=-1) > 4)  # in every row, whatever the right one was off by


@pytest.mark.parametrize("L", [2, 100])
def test_a_key_at_the_next_position_is_past_the_bound(L):
    w, norms, x, k, v = case(L)
    want, bound, _, _ = keys_and_values(w, norms, x, KV, np.arange(L) + 1)
    assert cached(k, *keys_and_values(w, norms, x, KV)[:2]) <= 1
    for j in range(L):
        assert cached(k[j], want[j], bound[j]) > 4
