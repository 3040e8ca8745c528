"""The order of keys where 64-bit scores tie or a group's sum is no number."""
import numpy as np
import pytest

from bybylang_amd import _abi, synth
from test_moe_gpu import F32, SIG, SOFT, routed

pytestmark = pytest.mark.gpu


def chosen(x, worth, groups, top_groups, k, keys):
    """The k best by `keys` in the groups that are worth most, ties to the lowest index."""
    size = len(x) // groups
    kept = sorted(range(groups), key=lambda i: (-worth[i], i))[:top_groups]
    pool = [e for i in kept for e in range(i * size, (i + 1) * size)]
    return sorted(pool, key=lambda e: (-keys[e], e))[:k]


@pytest.mark.parametrize("E,groups,top_groups", [(32, 4, 2), (96, 3, 2), (256, 8, 4), (60, 4, 3)])
@pytest.mark.parametrize("score", [SOFT, SIG])
def test_without_a_bias_logits_are_the_keys(hip, E, groups, top_groups, score):
    """Sigmoids of 40 and 60 are both 1 in 64 bits, softmax scores 800 below the largest both 0; groups by their two best do not make them alike."""
    g = synth.rng(E)
    size, k = E // groups, 7
    x = (40 + 20 * g.random((5, E))).astype(np.float32)
    if score == SIG:
        x[:, :size] -= 100
    else:
        x[:, 0] = 900
    ids, _ = routed(hip, x, F32, k, score=score, groups=groups, top_groups=top_groups, group_by=2)
    with np.errstate(over="ignore"):
        for t, row in enumerate(x.astype(np.float64)):
            s = 1 / (1 + np.exp(-row)) if score == SIG else np.exp(row - row.max()) / np.exp(row - row.max()).sum()
            worth = [np.sort(s[i * size:(i + 1) * size])[-2:].sum() for i in range(groups)]
            assert ids[t].tolist() == chosen(row, worth, groups, top_groups, k, row), t


@pytest.mark.parametrize("E,groups,top_groups", [(32, 4, 2), (60, 4, 2)])
def test_a_row_with_a_nan_keeps_different_experts(hip, E, groups, top_groups):
    g = synth.rng(E)
    x = g.integers(-2, 3, (6, E)).astype(np.float32)
    x[:, 5] = np.nan
    for bias in (None, np.zeros(E, np.float32)):
        for score in (SOFT, SIG):
            ids, _ = routed(hip, x, F32, 7, score=score, bias=bias, groups=groups, top_groups=top_groups, group_by=2)
            assert all(len(set(r)) == 7 and min(r) >= 0 and max(r) < E for r in ids.tolist())


@pytest.mark.parametrize("E,groups", [(32, 4), (60, 4), (256, 8)])
@pytest.mark.parametrize("at", [0, 1, 3])
def test_a_group_of_both_infinities(hip, E, groups, at):
    """A bias that holds +infinity beside -infinity makes a group's sum NaN: that group comes last, and no group more than asked for takes part."""
    g = synth.rng(E + at)
    size, k = E // groups, 6
    b = (0.3 * g.standard_normal(E)).astype(np.float32)
    b[at * size:(at + 1) * size] = -np.inf
    b[at * size + 2] = np.inf
    x = g.standard_normal((9, E)).astype(np.float32)
    ids, _ = routed(hip, x, F32, k, score=SIG, bias=b, groups=groups, top_groups=2, group_by=2)
    for t, row in enumerate(x.astype(np.float64)):
        key = 1 / (1 + np.exp(-row)) + b
        worth = [-np.inf if i == at else np.sort(key[i * size:(i + 1) * size])[-2:].sum() for i in range(groups)]
        assert ids[t].tolist() == chosen(row, worth, groups, 2, k, key), t
