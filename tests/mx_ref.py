"""Microscaled rows, routing and experts in 64 bits: what the GPU tests compare with.

A rounding to e4m3 is off by at most 2^-4 of the value, or 2^-10 times the scale below the least normal value 2^-6; one to
e2m1 by at most 2^-2 of the value (half a step of 0.5 at 1), or a quarter of the scale below 1.
"""
import numpy as np

from bybylang_amd import _abi

MX8, MX4 = _abi.MXFP8_KM, _abi.MXFP4_KM
MOST = {MX8: 448.0, MX4: 6.0}
DIGITS = {MX8: 3, MX4: 1}       # bits after the leading one
LEAST = {MX8: -6, MX4: 0}       # exponent of the least normal value


def row_bytes(K, fmt):
    return K if fmt == MX8 else K // 2


def scale_bytes(amax, fmt):
    """Scale bytes of groups with these largest magnitudes (float64, exact for fp32 inputs)."""
    amax = np.asarray(amax, np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.floor(np.log2(amax)) - np.log2(2.0 ** np.floor(np.log2(MOST[fmt])))
    e = np.where(np.isfinite(e), e, -200).astype(np.int64)
    for _ in range(2):  # the logarithm may be off by one at a power of two
        e = np.where(amax > MOST[fmt] * 2.0 ** np.clip(e, -300, 300), e + 1, e)
        e = np.where(amax <= MOST[fmt] * 2.0 ** np.clip(e - 1, -300, 300), e - 1, e)
    return np.where(np.isfinite(amax), np.maximum(e + 127, 0), 255).astype(np.uint8)


def nearest(z, fmt):
    """z to the format's nearest value, ties to even."""
    with np.errstate(divide="ignore"):
        grid = 2.0 ** (np.maximum(np.floor(np.log2(np.abs(z))), LEAST[fmt]) - DIGITS[fmt])
    return np.round(z / grid) * grid


def codes_of(z, fmt):
    """Bits of values that the format holds exactly."""
    a, sign = np.abs(z), np.signbit(z).astype(np.uint8)
    d, least = DIGITS[fmt], LEAST[fmt]
    with np.errstate(divide="ignore"):
        e = np.where(a >= 2.0 ** least, np.floor(np.log2(np.where(a > 0, a, 1))), least - 1)
    man = np.where(e >= least, a / 2.0 ** e - 1, a / 2.0 ** least) * 2 ** d
    bits = ((e - least + 1).astype(np.int64) << d) + man.astype(np.int64)
    return (bits + (sign.astype(np.int64) << (7 if fmt == MX8 else 3))).astype(np.uint8)


def km(a):
    """[R, K] in element order -> memory order."""
    R, K = a.shape
    return np.ascontiguousarray(a.reshape(R, K // 32, 2, 16).transpose(0, 1, 3, 2)).reshape(R, K)


def from_km(a):
    R, K = a.shape
    return np.ascontiguousarray(a.reshape(R, K // 32, 16, 2).transpose(0, 1, 3, 2)).reshape(R, K)


def quantize(v, fmt):
    """float [R, K] -> (the buffer's bytes, the float64 rows they stand for)."""
    v = np.asarray(v, np.float64)
    R, K = v.shape
    g = v.reshape(R, K // 32, 32)
    amax = np.abs(g).max(2) if K else np.zeros((R, 0))
    amax = np.where(np.isnan(g).any(2), np.nan, amax)
    s = scale_bytes(amax, fmt)
    f = 2.0 ** (s.astype(np.float64) - 127)
    z = np.where((s == 255)[..., None], 0.0, nearest(np.where(np.isfinite(g), g, 0.0) / f[..., None], fmt))
    codes = km(codes_of(z.reshape(R, K), fmt))
    if fmt == MX4:
        codes = codes[:, 0::2] | codes[:, 1::2] << 4
    rows = np.where((s == 255)[..., None], np.nan, z * f[..., None]).reshape(R, K)
    return np.concatenate([codes.reshape(-1), s.reshape(-1)]), rows


def parts(buf, R, K, fmt):
    """(values [R, K] float64 in element order, scale bytes [R, K / 32]) of a buffer."""
    n = R * row_bytes(K, fmt)
    b, s = np.asarray(buf[:n]).reshape(R, -1), np.asarray(buf[n:n + R * K // 32]).reshape(R, K // 32)
    if fmt == MX4:
        b = np.stack([b & 15, b >> 4], -1).reshape(R, K)
    d = DIGITS[fmt]
    body = b & (127 if fmt == MX8 else 7)
    e, man = body >> d, body & (2 ** d - 1)
    v = np.where(e > 0, (1 + man / 2.0 ** d) * 2.0 ** (e.astype(float) - 1 + LEAST[fmt]), man / 2.0 ** d * 2.0 ** LEAST[fmt])
    return from_km(np.where(b >> (7 if fmt == MX8 else 3), -v, v)), s


def rows(buf, R, K, fmt):
    """The float64 rows of a buffer (NaN in groups whose scale is)."""
    v, s = parts(buf, R, K, fmt)
    f = np.where(s == 255, np.nan, 2.0 ** (s.astype(np.float64) - 127))
    return (v.reshape(R, K // 32, 32) * f[..., None]).reshape(R, K)


def close_mx(buf, want, slack, fmt, what=""):
    """A buffer against the float64 rows that were rounded into it, each known within `slack`: every scale is that of some largest magnitude
    in reach, and every value within half a step and the slack."""
    R, K = want.shape
    v, s = parts(buf, R, K, fmt)
    slack = np.broadcast_to(slack, want.shape)
    g, sl = want.reshape(R, K // 32, 32), slack.reshape(R, K // 32, 32)
    lo = scale_bytes(np.maximum(np.abs(g) - sl, 0).max(2), fmt)
    hi = scale_bytes((np.abs(g) + sl).max(2), fmt)
    assert np.all((s >= lo) & (s <= hi)), f"{what}: scales off at {np.argwhere((s < lo) | (s > hi))[:4].tolist()}"
    f = np.repeat(2.0 ** (s.astype(np.float64) - 127), 32, axis=1)
    half = {MX8: np.maximum(2.0 ** -4 * (np.abs(want) + slack), 2.0 ** -10 * f), MX4: np.maximum(0.25 * (np.abs(want) + slack), 0.25 * f)}[fmt]
    off = np.abs(v * f - want)
    bad = ~(off <= half + slack)
    assert not bad.any(), f"{what}: {bad.sum()} of {off.size} off, worst {np.max(off / (half + slack)):.3g} of the bound"


def random_rows(g, R, K, fmt, spread=2):
    """Rows whose groups differ in size: (buffer, float64 rows)."""
    v = g.standard_normal((R, K)) * 2.0 ** g.integers(-spread, spread + 1, (R, K // 32)).repeat(32, axis=1)
    return quantize(v.astype(np.float32), fmt)


def silu(v):
    with np.errstate(over="ignore"):
        return v / (1 + np.exp(-v))


def plan(ids, experts):
    """(offsets, order) of assignments [T, k]."""
    flat = np.asarray(ids).reshape(-1)
    order = [a for e in range(experts) for a in np.flatnonzero(flat == e)]
    return np.concatenate([[0], np.cumsum([(flat == e).sum() for e in range(experts)])]).astype(np.int32), np.array(order, np.int32)


def route(logits, bias, k, score, groups, top_groups, group_by, renorm, scale):
    """(ids, weights) of float64 logits [T, E]: the router's definition, token by token."""
    T, E = logits.shape
    ids, weights = np.zeros((T, k), np.int32), np.zeros((T, k))
    for t in range(T):
        x = logits[t]
        with np.errstate(invalid="ignore", over="ignore"):
            if score == _abi.MOE_SIGMOID:
                s = 1 / (1 + np.exp(-x))
            elif np.isnan(x).any():
                s = np.full(E, np.nan)
            elif x.max() == -np.inf:
                s = np.zeros(E)
            else:
                z = np.exp(np.where(x == x.max(), 0.0, x - x.max()))
                s = z / z.sum()
        key = x if bias is None and not (groups > 1 and group_by == 2) else s + (0 if bias is None else bias)
        rank = np.where(np.isnan(key), -np.inf, key)
        pool = range(E)
        if groups > 1:
            size = E // groups
            worth = [sum(sorted(rank[i * size:(i + 1) * size])[-group_by:]) for i in range(groups)]
            pool = [e for i in sorted(range(groups), key=lambda i: (-worth[i], i))[:top_groups] for e in range(i * size, (i + 1) * size)]
        ids[t] = sorted(pool, key=lambda e: (np.isnan(key[e]), -rank[e], e))[:k]
        w = s[ids[t]]
        if renorm:
            w = np.zeros(k) if w.sum() == 0 else w / w.sum()
        weights[t] = w * scale
    return ids, weights
