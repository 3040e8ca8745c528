"""byhip_rope_steps, the host helper that turns a base and a scaling into turns per position (no GPU)."""
import numpy as np
import pytest

from bybylang_amd import _abi
from bybylang_amd import device as dev


def turns(steps):
    return steps.astype(np.float64) / 2.0**64


def freqs(r, base=10000.0):
    return base ** (-np.arange(0, r, 2) / r) / (2 * np.pi)


# 2^-64 of a turn and the double's own rounding, relative to the frequency
def same(got, want):
    assert np.all(np.abs(turns(got) - want) <= 2.0**-64 + 2.0**-50 * want)


@pytest.mark.parametrize("r", [2, 64, 80, 128, 256])
def test_plain_and_linear(r):
    s, m = dev.rope_steps(r)
    same(s, freqs(r))
    assert m == 1.0
    s, m = dev.rope_steps(r, scaling=dev.ROPE_LINEAR, factor=8.0)
    same(s, freqs(r) / 8)
    assert m == 1.0


def test_base_slows_the_slowest_pair_by_the_factor():
    s, _ = dev.rope_steps(128, 5e5, dev.ROPE_BASE, 4.0)
    want = freqs(128, 5e5 * 4.0 ** (128 / 126))
    same(s, want)
    assert want[0] == freqs(128, 5e5)[0]
    assert abs(want[-1] * 4 / freqs(128, 5e5)[-1] - 1) < 1e-12


def test_parts():
    s, m = dev.rope_steps(128, 1e4, dev.ROPE_PARTS, 8.0, 4096, 1.0, 32.0)
    f = freqs(128)
    keep = np.clip((4096 * f - 1) / 31, 0, 1)
    same(s, f / 8 * (1 - keep) + f * keep)
    assert m == np.float32(0.1 * np.log(8.0) + 1)
    assert keep[0] == 1 and keep[-1] == 0


def test_nothing_rotated():
    s, m = dev.rope_steps(0)
    assert s.size == 0 and m == 1.0


@pytest.mark.parametrize("args,match", [
    ((7,), "not even"),
    ((-2,), "not even"),
    ((64, 1.0), "rotary base"),
    ((64, float("nan")), "rotary base"),
    ((64, 1e4, 9), "rotary scaling 9"),
    ((64, 1e4, 1, 0.5), "scaling factor"),
    ((64, 1e4, 3, 2.0, 0.0), "positions"),
    ((64, 1e4, 3, 2.0, 4096.0, 4.0, 2.0), "turns"),
])
def test_refusals(args, match):
    with pytest.raises(_abi.HipBackendError, match=match):
        dev.rope_steps(*args)
    assert _abi.load().byhip_rope_steps(64, 1e4, 0, 1.0, 0.0, 1.0, 32.0, None, None) == _abi.BYHIP_ERROR
