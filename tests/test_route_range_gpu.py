"""Renormalised weights where every chosen score is next to nothing or vanishes in fp32: sigmoids of very negative logits, softmax scores of experts that a
bias chose far below the row's largest logit. Bounds as in test_moe_gpu.py."""
import numpy as np
import pytest

from bybylang_amd import _abi, synth
from paged_ref import to_bits
from test_moe_gpu import F16, F32, SIG, SOFT, check_route, routed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E,k", [(1, 1), (12, 1), (40, 8), (200, 8), (300, 70)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dt", [F32, F16])
def test_sigmoids_far_down(hip, E, k, bias, dt):
    """Rows around -60 (whose 1 / sum fits fp32), -88, -91, -95, -100, -120, -300, -700 and, for one, of a single logit near 0 among them."""
    g = synth.rng(E)
    x = g.standard_normal((9, E)) + np.array([-60, -88, -91, -95, -100, -120, -300, -700, -100])[:, None]
    x[8, E // 2] = -0.5
    check_route(hip, 9, E, k, dt=dt, seed=k, x=to_bits(x, dt), score=SIG, bias=bias, scale=2.5)


@pytest.mark.parametrize("E,k", [(40, 2), (40, 8), (300, 70)])
@pytest.mark.parametrize("groups", [1, 4])
def test_softmax_chosen_by_the_bias(hip, E, k, groups):
    """The bias chooses experts 90, 110 and up to 600 below the row's largest logit."""
    T, half = 6, E // 2
    g = synth.rng(k)
    x = g.standard_normal((T, E)).astype(np.float32)
    x[:, :half] += np.array([0, 90, 110, 150, 400, 600], np.float32)[:, None]
    b = np.zeros(E, np.float32)
    b[half:] = 5 + g.random(E - half).astype(np.float32)
    from mx_ref import route
    ids, w = routed(hip, x, F32, k, score=SOFT, bias=b, groups=groups, top_groups=groups // 2 or 1, group_by=1)
    want_ids, want = route(x.astype(np.float64), b.astype(np.float64), k, SOFT, groups, groups // 2 or 1, 1, True, 1.0)
    assert np.array_equal(ids, want_ids) and np.all(ids >= half)
    # exp's argument is formed in 64 bits; a rounding of each share, their sum (k terms), the quotient and the product
    assert np.all(np.abs(w - want) <= (k + 8) * 2.0**-24 * want + 2.0**-126)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("score", [SOFT, SIG])
def test_masked_rows_have_no_weights(hip, bias, score):
    """Rows of a mask's value (-infinity, the types' lowest, -1e9, -1000) have weights 0 as sigmoids; as a softmax all but -infinity are rows like any."""
    E, k = 24, 3
    for value in (-np.inf, np.finfo(np.float32).min, -65504.0, -1e9, -1000.0):
        x = np.full((2, E), value, np.float32)
        x[1, 3] = 1.0
        b = np.linspace(0, 0.5, E).astype(np.float32) if bias else None
        ids, w = routed(hip, x, F32, k, score=score, bias=b)
        if score == SIG or value == -np.inf:
            assert np.all(w[0] == 0)
        else:
            assert np.all(np.abs(w[0] - 1 / 3) <= 5 * 2.0**-24)
        assert np.array_equal(w[1], np.where(ids[1] == 3, 1, 0))


def test_nan_is_not_taken_for_nothing(hip):
    x = np.full((2, 8), -np.inf, np.float32)
    x[0, 5] = x[1] = np.nan
    for score in (SOFT, SIG):
        _, w = routed(hip, x, F32, 8, score=score)
        assert np.isnan(w).all()
