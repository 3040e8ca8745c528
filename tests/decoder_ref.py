"""One attention block over a paged cache in 64 bits, in the two halves that the cache separates: the keys and values that belong in
it, and the block's rows given what it holds. So no bound has to allow for the cache's 16 bits, and a row, key or position out
of place shows.

Bounds. A product of K terms: the matmuls hold 22 bits and more of both operands and add up in fp32, so an error of deviation
(2^-23 sqrt 2 + 2^-24 sqrt K) of the root of the terms' squares, taken 6 times (tens of thousands of values are compared); its input, a norm's row,
is off by up to 2^-18 as a whole. Rotary positions mix two values: their errors add, and 5e-7 of both. Scores, weights and sums
as in the tests of attention alone: 2 sqrt(D) 2^-24 of sum |q k|, 4e-6, sqrt(L) 2^-22."""
import numpy as np

EPS = 1e-5


def product(x, w):
    """x @ w and its bound."""
    s = (2.0**-22.5 + 2.0**-24 * np.sqrt(x.shape[1])) * np.sqrt((x * x) @ (w * w))
    y = x @ w
    return y, 6 * s


def rotated(x, pos):
    """Rotary positions over halves, base 10000."""
    half = x.shape[-1] // 2
    angle = pos[:, None] * 10000.0 ** (-np.arange(half) / half)
    c, s = np.cos(angle)[:, None, :], np.sin(angle)[:, None, :]
    a, b = x[..., :half], x[..., half:]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def rotated_bound(x, e):
    half = x.shape[-1] // 2
    both = e[..., :half] + e[..., half:] + 5e-7 * (np.abs(x[..., :half]) + np.abs(x[..., half:]))
    return np.concatenate([both, both], -1)


def normed(x, gamma):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * gamma


def heads_of(y, w, heads):
    x, e = product(y, w)
    return x.reshape(len(x), heads, -1), (e + 2.0**-18 * np.abs(x)).reshape(len(x), heads, -1)


def keys_and_values(w, norms, x, kv, pos=None):
    """(keys, bound, values, bound) of a sequence's rows x, before the cache rounds them."""
    y = normed(x.astype(np.float64), norms[0])
    k, ek = heads_of(y, w[1], kv)
    v, ev = heads_of(y, w[2], kv)
    pos = np.arange(len(x)) if pos is None else pos
    return rotated(k, pos), rotated_bound(k, ek), v, ev


def cached(got, want, bound):
    """Worst share of the bound between the fp16 values of a cache and what belongs there."""
    return np.max(np.abs(got - want) / (2.0**-11 * (np.abs(want) + bound) + 2.0**-25 + bound), initial=0.0)


def rows_of(w, norms, x, k, v, n, heads, turn=0, share=1.0, drop=0):
    """(the block's last n rows, bound) over the cache's keys and values k, v [L, kv, D] of a sequence whose rows are x. turn, share,
    drop: planted mistakes (queries turned too far, part of the attention, last keys not read)."""
    L, kv, D = k.shape
    x = x[L - n:].astype(np.float64)
    pos = np.arange(L - n, L)
    q, eq = heads_of(normed(x, norms[0]), w[0], heads)
    q, eq = rotated(q, pos + turn), rotated_bound(q, eq)
    a, ea = np.zeros((n, heads, D)), np.zeros((n, heads, D))
    seen = np.arange(L)[None, :] <= pos[:, None] - drop
    for h in range(heads):
        kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
        s = np.where(seen, q[:, h] @ kh.T * D**-0.5, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        off = (np.sqrt((eq[:, h] ** 2) @ (kh * kh).T) + 2 * np.sqrt(D) * 2.0**-24 * (np.abs(q[:, h]) @ np.abs(kh).T)) * D**-0.5
        off = np.where(seen, off, 0).max(-1) + 4e-6 + np.sqrt(L) * 2.0**-22
        a[:, h] = p @ vh
        ea[:, h] = off[:, None] * (p @ np.abs(vh) + np.abs(a[:, h]))
    a, ea = share * a.reshape(n, -1), ea.reshape(n, -1)
    o, eo = product(a, w[3])
    h = x + o
    eh = eo + ea @ np.abs(w[3]) + 2.0**-22 * np.abs(h)
    rms = np.sqrt((h * h).mean(-1, keepdims=True) + EPS)
    y = h / rms * norms[1]
    return y, (eh * np.abs(norms[1]) + np.abs(y) * np.sqrt((eh * eh).mean(-1, keepdims=True))) / rms + 2.0**-18 * np.abs(y)
