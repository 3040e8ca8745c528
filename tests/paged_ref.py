"""The operators over a paged cache in 64 bits, sequence by sequence: what the GPU tests compare with."""
import numpy as np

from bybylang_amd import _abi

UNIT = {_abi.F32: 2.0**-24, _abi.F16: 2.0**-11, _abi.BF16: 2.0**-8}   # half a unit in the last place, relative
TINY = {_abi.F32: 2.0**-149, _abi.F16: 2.0**-25, _abi.BF16: 2.0**-134}


def to_bits(a, dtype):
    """float array -> the dtype's array as numpy keeps it (bf16: uint16 bits, nearest even)."""
    a = np.ascontiguousarray(a, np.float32)
    if dtype == _abi.F32:
        return a
    if dtype == _abi.F16:
        return a.astype(np.float16)
    u = a.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    nan = np.isnan(a)
    r[nan] = (u[nan] >> 16).astype(np.uint16) | 0x40
    return r


def from_bits(a, dtype):
    """The dtype's array -> float64."""
    if dtype == _abi.BF16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def rounded(a, dtype):
    return from_bits(to_bits(a, dtype), dtype)


def close(got, want, dtype, slack, what=""):
    """|got - want| <= slack (fp32 arithmetic, absolute) + the dtype's rounding; NaN and infinities agree."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN in other places"
    inf = ~fine & ~np.isnan(want)
    assert np.array_equal(got[inf], want[inf]), f"{what}: infinities differ"
    slack = np.broadcast_to(slack, want.shape)[fine]
    off = np.abs(got[fine] - want[fine])
    bound = slack + UNIT[dtype] * (np.abs(want[fine]) + slack) + TINY[dtype]
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} of {off.size} off, worst {np.max(off / bound):.3g} of the bound"


def paged(g, lens, page, pages, extra_cols=0):
    """Page tables [len(lens)][stride] over distinct random pages, -1 where a sequence holds none."""
    need = [-(-n // page) for n in lens]
    assert sum(need) <= pages
    t = np.full((len(lens), max(need + [1]) + extra_cols), -1, np.int32)
    ids = g.permutation(pages).astype(np.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = ids[at:at + n]
        at += n
    return t


def rope(x, pos, steps, rot, layout, magnitude):
    """x [n, heads, dim] float64 turned by its positions."""
    y = x.copy()
    turns = (np.asarray(pos, np.uint64)[:, None] * np.asarray(steps, np.uint64)[None, :]).astype(np.float64) / 2.0**64
    z = np.exp(2j * np.pi * turns)[:, None, :] * magnitude
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == _abi.ROPE_HALVES else (slice(0, rot, 2), slice(1, rot, 2))
    w = (x[..., a] + 1j * x[..., b]) * z
    y[..., a], y[..., b] = w.real, w.imag
    return y


def visible(L, n, window, prefix):
    """[n, L]: which keys each row sees."""
    p = (L - n + np.arange(n))[:, None]
    j = np.arange(L)[None, :]
    see = j <= p
    if window > 0:
        see &= p - j < window
    return see | (j < prefix)


def attention(q, k, v, scale, cap, window, slopes, prefix, seen=None):
    """q [n, H, D], k and v [L, Hk, D] float64 -> (out [n, H, D], and for bounds: the weighted mean of |v|, the
    largest sum of |q_d k_d| * scale among the seen keys and the mean of |v| over 1 / sum of weights times their
    number). Hidden keys have no part, whatever they hold."""
    n, H, D = q.shape
    L, Hk, _ = k.shape
    see = visible(L, n, window, prefix)
    if seen is not None:
        see = see & seen[None, :]
    out, mean, flat = np.zeros((n, H, D)), np.zeros((n, H, D)), np.zeros((n, H, D))
    size = np.zeros((n, H, 1))
    dist = np.abs((L - n + np.arange(n))[:, None] - np.arange(L)[None, :])
    for h in range(H):
        kh, vh = k[:, h // (H // Hk)], v[:, h // (H // Hk)]
        with np.errstate(invalid="ignore", over="ignore"):
            s = (q[:, h] @ kh.T) * scale
            big = (np.abs(q[:, h]) @ np.abs(kh).T) * abs(scale)
            if cap > 0:
                s = cap * np.tanh(s / cap)
            if slopes is not None:
                s = s - slopes[h] * dist
        for i in range(n):
            at = np.flatnonzero(see[i])
            if at.size == 0:
                continue
            si = s[i, at]
            m = np.max(si)
            if m == -np.inf:
                continue
            with np.errstate(invalid="ignore"):
                w = np.exp(si - m)
                out[i, h] = (w @ vh[at]) / w.sum()
                mean[i, h] = (w @ np.abs(vh[at])) / w.sum()
                flat[i, h] = np.abs(vh[at]).sum(0) / w.sum()
                size[i, h] = np.max(big[i, at])
    return out, mean, size, flat


def norm(v, kind, eps, weight=None, bias=None):
    mean = v.mean(1, keepdims=True) if kind == _abi.NORM_LAYER else 0.0
    d = v - mean
    y = d / np.sqrt((d * d).mean(1, keepdims=True) + eps)
    if weight is not None:
        y = y * weight
    return y if bias is None else y + bias
