"""Performance cases of the attention half of a decoder layer over a paged cache: what a serving program
calls between the quantized projections, per operator and regime.

Kinds
  rope   rope_append: rotary positions on the query and key heads of QKV rows, the keys and values
         written to their pages.
  attn   paged_attention: rows of new tokens (one, a chunk, or a mixed batch) over a paged cache, with
         grouped heads, a tanh cap, a sliding window, a bias by distance and an open prefix.
  fork   cache_fork and cache_grow: sequences continue others, share their pages and get room for the next
         token (a last page that is only partly filled is copied).
  compact  cache_compact: live pages move to the front of the pool.
  norm   norm_block: the norm after a block, its gate, the scaled residual and the norm before the next.

A cache is [pages][kv_heads][page][dim] for keys and the same for values. Row i of a sequence that brings n
tokens to a length L has position L - n + i.
"""
import math

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
CODE = {"f32": 0, "f16": 1, "bf16": 2}


def listed():
    return [
        # one decode step of 32 sequences, the session's fp32 QKV rows, whole heads
        {"name": "rope_decode", "kind": "rope", "batch": 32, "n_lo": 1, "n_hi": 1, "len_lo": 60, "len_hi": 2000, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "dtype": "f16", "io": "f32", "rot": 128, "layout": "half", "scaling": "none"},
        # three prompts of no round length, neighbouring pairs, half of each head turned, scaled for a long context
        {"name": "rope_prompts", "kind": "rope", "batch": 3, "n_lo": 701, "n_hi": 2111, "len_lo": 2500, "len_hi": 9001, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bf16", "io": "bf16", "rot": 64, "layout": "pairs", "scaling": "parts"},
        # one token of one short sequence: latency
        {"name": "attn_one", "kind": "attn", "batch": 1, "n_lo": 1, "n_hi": 1, "singles": 1, "len_lo": 777, "len_hi": 777, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "dtype": "f16", "io": "f16", "cap": 0.0, "window": 0, "slopes": False, "prefix": 0},
        # one decode step of 64 sequences of many lengths
        {"name": "attn_decode", "kind": "attn", "batch": 64, "n_lo": 1, "n_hi": 1, "singles": 64, "len_lo": 300, "len_hi": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bf16", "io": "bf16", "cap": 0.0, "window": 0, "slopes": False, "prefix": 0},
        # two long contexts, one token each, at the session's fp32
        {"name": "attn_long", "kind": "attn", "batch": 2, "n_lo": 1, "n_hi": 1, "singles": 2, "len_lo": 100001, "len_hi": 131072, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "f16", "io": "f32", "cap": 0.0, "window": 0, "slopes": False, "prefix": 0},
        # a chunk of a long prompt over what is cached of it
        {"name": "attn_chunk", "kind": "attn", "batch": 1, "n_lo": 4096, "n_hi": 4096, "singles": 0, "len_lo": 16384, "len_hi": 16384, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bf16", "io": "bf16", "cap": 0.0, "window": 0, "slopes": False, "prefix": 0},
        # a serving batch: prompt chunks beside decoding sequences, capped scores in a window, smaller heads
        {"name": "attn_mixed", "kind": "attn", "batch": 24, "n_lo": 90, "n_hi": 700, "singles": 18, "len_lo": 700, "len_hi": 4001, "heads": 24, "kv_heads": 8, "dim": 64,
         "page": 16, "dtype": "f16", "io": "f16", "cap": 30.0, "window": 1024, "slopes": False, "prefix": 0},
        # prompts with an open prefix and a bias by distance at the session's fp32, heads of no power of two
        {"name": "attn_prefix", "kind": "attn", "batch": 3, "n_lo": 130, "n_hi": 509, "singles": 0, "len_lo": 600, "len_hi": 2045, "heads": 12, "kv_heads": 4, "dim": 80,
         "page": 32, "dtype": "bf16", "io": "f32", "cap": 0.0, "window": 0, "slopes": True, "prefix": 200},
        # a step of 4 beams each of 4 prompts: every beam continues a parent and gets room for a token
        {"name": "fork_beams", "kind": "fork", "parents": 4, "children": 16, "len_lo": 500, "len_hi": 2001, "add": 1, "layers": 4, "pages": 512, "kv_heads": 8, "dim": 128,
         "page": 32, "dtype": "f16"},
        # a fragmented pool, half of it live
        {"name": "compact_pool", "kind": "compact", "slots": 48, "len_lo": 100, "len_hi": 2000, "live": 0.5, "layers": 4, "kv_heads": 8, "dim": 128,
         "page": 32, "dtype": "bf16"},
        # the residual stream of one decode step of 32 sequences
        {"name": "norm_decode", "kind": "norm", "rows": 32, "cols": 4096, "x": "f32", "h": "f32", "y": "f16", "post": "rms", "pre": "rms", "gate": False, "scale": 1.0},
        # the residual stream of a prompt, gated, layer norms
        {"name": "norm_prompt", "kind": "norm", "rows": 4099, "cols": 5120, "x": "bf16", "h": "f32", "y": "bf16", "post": "layer", "pre": "layer", "gate": True, "scale": 0.7},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the listed ones' ranges, at most the largest one's work."""
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= 9.4e8 and w["flops"] <= 9.5e11 and _scores(case) <= 2.2e9:
            return case


def _scores(c):
    """Scores of the plain form, which pads every sequence to the longest."""
    return c["batch"] * c["heads"] * max(_new(c)) * max(_lens(c)) if c["kind"] == "attn" else 0


def _heads(rng):
    dim = rng.choice([64, 80, 112, 128, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8, 8])
    return {"heads": kv * rng.choice([1, 2, 4, 4, 5, 7, 8]), "kv_heads": kv, "dim": dim, "page": rng.choice([16, 16, 32, 64, 128, 40]), "dtype": rng.choice(["f16", "bf16"])}


def _draw(rng):
    kind = rng.choice(["rope", "attn", "attn", "attn", "fork", "compact", "norm"])
    if kind == "norm":
        gate, x = rng.random() < 0.5, rng.choice(["f32", "f16", "bf16"])
        cols = _log(rng, 80, 16384)
        return {"kind": kind, "rows": _log(rng, 1, 8192), "cols": cols if rng.random() < 0.3 else cols // 80 * 80, "x": x, "h": rng.choice(["f32", x]),
                "y": rng.choice(["f16", "bf16", x]), "post": rng.choice(["rms", "layer", "none"]), "pre": rng.choice(["rms", "layer"]), "gate": gate, "scale": rng.choice([1.0, 0.5])}
    h = _heads(rng)
    if kind == "fork":
        parents = _log(rng, 1, 16)
        hi = _log(rng, 64, 2001)
        children = parents * _log(rng, 1, 8)
        return {"kind": kind, "parents": parents, "children": children, "len_lo": max(1, hi // 3), "len_hi": hi, "add": _log(rng, 1, 100), "layers": rng.randint(1, 6),
                "pages": parents * (hi // h["page"] + 1) + children * (2 + 100 // h["page"] + 1) + rng.randint(1, 200), "kv_heads": h["kv_heads"], "dim": h["dim"], "page": h["page"],
                "dtype": h["dtype"]}
    if kind == "compact":
        hi = _log(rng, 64, 2000)
        return {"kind": kind, "slots": _log(rng, 4, 64), "len_lo": max(1, hi // 9), "len_hi": hi, "live": round(rng.uniform(0.3, 0.9), 2), "layers": rng.randint(1, 4),
                "kv_heads": h["kv_heads"], "dim": h["dim"], "page": h["page"], "dtype": h["dtype"]}
    batch = _log(rng, 1, 64)
    hi = _log(rng, 200, 16384 if batch > 4 else 131072)
    c = {"kind": kind, "batch": batch, "len_lo": max(1, hi // rng.choice([1, 2, 8])), "len_hi": hi, **h, "io": rng.choice([h["dtype"], h["dtype"], "f32"])}
    if kind == "rope":
        n = min(hi, _log(rng, 1, 2000))
        return {**c, "n_lo": max(1, n // 3), "n_hi": n, "rot": rng.choice([h["dim"], h["dim"], h["dim"] // 2]), "layout": rng.choice(["half", "pairs"]),
                "scaling": rng.choice(["none", "linear", "parts"])}
    singles = rng.choice([batch, batch, 0, rng.randint(0, batch)])
    n = 1 if singles == batch else min(hi, _log(rng, 2, 4096))
    return {**c, "n_lo": max(1, n // 3), "n_hi": n, "singles": singles, "cap": rng.choice([0.0, 0.0, 20.0, 50.0]), "window": rng.choice([0, 0, 0, _log(rng, 16, 4096)]),
            "slopes": rng.random() < 0.25, "prefix": rng.choice([0, 0, 0, _log(rng, 1, 500)])}


# ── sizes ───────────────────────────────────────────────────────────────────────────────────


def _spread(lo, hi, count):
    """`count` sizes spread over lo..hi, the largest first."""
    return [hi if i == 0 else lo + int((hi - lo) * ((0.61803399 * i) % 1.0)) for i in range(count)]


def _lens(c):
    return _spread(c["len_lo"], c["len_hi"], c["batch"])


def _new(c):
    many = c["batch"] - c.get("singles", 0)
    n = _spread(c["n_lo"], c["n_hi"], many) + [1] * (c["batch"] - many)
    return [min(a, b) for a, b in zip(n, _lens(c))]


def _visible(c):
    """(pairs of a row and a key that it sees, keys that some row sees) over all sequences."""
    pairs = keys = 0
    for n, L in zip(_new(c), _lens(c)):
        p = np.arange(L - n, L, dtype=np.int64)
        lo = np.maximum(0, p + 1 - c["window"]) if c["window"] else np.zeros_like(p)
        pre = min(c["prefix"], L)
        over = np.maximum(0, np.minimum(pre, p + 1) - lo)
        pairs += int((p + 1 - lo + pre - over).sum())
        keys += L - max(int(lo[0]), pre) + pre if pre < L else L
    return pairs, keys


def work(c):
    k = c["kind"]
    if k == "norm":
        n = c["rows"] * c["cols"]
        return {"bytes": n * (SIZE[c["x"]] + 2 * SIZE[c["h"]] + SIZE[c["y"]]) + 4 * c["cols"] * 4, "flops": 16 * n}
    row = c["kv_heads"] * c["dim"] * SIZE[c["dtype"]]
    if k == "fork":
        copies = sum(1 for i in range(c["children"]) if _spread(c["len_lo"], c["len_hi"], c["parents"])[i % c["parents"]] % c["page"])
        ints = 8 * c["children"] * (c["len_hi"] // c["page"] + 2)
        return {"bytes": copies * c["layers"] * 4 * row * c["page"] + ints, "flops": 0}
    if k == "compact":
        pages, held = _compact_sizes(c)
        return {"bytes": (1 - held / pages) * held * c["layers"] * 4 * row * c["page"] + 8 * (held + pages), "flops": 0}
    T = sum(_new(c))
    if k == "rope":
        return {"bytes": T * (c["heads"] + 2 * c["kv_heads"]) * c["dim"] * (SIZE[c["io"]] + SIZE[c["dtype"]]), "flops": 3 * T * (c["heads"] + c["kv_heads"]) * c["rot"]}
    pairs, keys = _visible(c)
    return {"bytes": 2 * keys * row + 2 * T * c["heads"] * c["dim"] * SIZE[c["io"]], "flops": 4 * pairs * c["heads"] * c["dim"]}


def _compact_sizes(c):
    """(pages of the pool, pages that sequences hold)."""
    held = sum(-(-n // c["page"]) for n in _spread(c["len_lo"], c["len_hi"], c["slots"]))
    return max(held + 1, int(held / c["live"])), held


# ── inputs ──────────────────────────────────────────────────────────────────────────────────


class Gen:
    """Seeded inputs on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)

    def normal(self, *shape, dtype="f32", scale=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda").mul_(scale).to(TORCH[dtype])

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda", dtype=torch.int32)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(g, lens, page, pages, extra=0):
    """Page tables of sequences of these lengths: pages of the pool in random order, -1 past the end."""
    need = [-(-n // page) for n in lens]
    width = max(need) + extra
    t = torch.full((len(lens), width), -1, dtype=torch.int32)
    ids, at = g.order(pages).cpu(), 0
    for b, n in enumerate(need):
        t[b, :n] = ids[at:at + n]
        at += n
    return t.cuda()


def _steps(rot, scaling):
    """Turns per position of each pair as a fraction of 2^64: frequencies 10000^(-2i/r) / 2 pi; for long
    contexts divided by 8 ("linear"), or by 8 only for the pairs that turn less than once in 4096 positions,
    with a ramp to those that turn 32 times ("parts", and then magnitude 0.1 ln 8 + 1)."""
    f = 10000.0 ** (-np.arange(0, rot, 2, dtype=np.float64) / rot) / (2 * np.pi)
    if scaling == "linear":
        f = f / 8
    if scaling == "parts":
        ramp = np.clip((4096 * f - 1) / (32 - 1), 0, 1)
        f = f / 8 * (1 - ramp) + f * ramp
    steps = np.array([int(x * 2.0**64) for x in f], dtype=np.uint64).view(np.int64)
    return torch.from_numpy(steps).cuda(), (0.1 * math.log(8) + 1) if scaling == "parts" else 1.0


def prepare(case, seed):
    """Inputs, the cache and its tables as a serving program holds them before the call."""
    c, g = case, Gen(seed)
    s = {"c": c}
    if c["kind"] == "norm":
        M, N = c["rows"], c["cols"]
        s["x"], s["res"] = g.normal(M, N, dtype=c["x"], scale=0.8), g.normal(M, N, dtype=c["h"], scale=2.0)
        for at in ("post", "pre"):
            s[at + "_w"] = 1 + g.normal(N, scale=0.2)
            s[at + "_b"] = g.normal(N, scale=0.1)
        s["gate"] = g.normal(N, scale=0.5) if c["gate"] else None
        s["h"], s["y"] = torch.empty(M, N, dtype=TORCH[c["h"]], device="cuda"), torch.empty(M, N, dtype=TORCH[c["y"]], device="cuda")
        return _ready(s)
    shape = (c["kv_heads"], c["page"], c["dim"])
    if c["kind"] == "fork":
        lens = _spread(c["len_lo"], c["len_hi"], c["parents"])
        t = _table(g, lens, c["page"], c["pages"], 1 + -(-c["add"] // c["page"]))
        s["table"] = torch.cat([t, torch.full((c["children"], t.shape[1]), -1, dtype=torch.int32, device="cuda")])
        s["lens"] = _ints(lens + [0] * c["children"])
        s["parents"] = _ints([i % c["parents"] for i in range(c["children"])])
        s["rows"] = _ints([c["parents"] + i for i in range(c["children"])])
        s["add"] = _ints([c["add"]] * c["children"])
        s["kv"] = g.normal(c["layers"], 2, c["pages"], *shape, dtype=c["dtype"])
        s["refs"] = _refs(s["table"], c["pages"])
    elif c["kind"] == "compact":
        lens = _spread(c["len_lo"], c["len_hi"], c["slots"])
        pages, _ = _compact_sizes(c)
        s["table"], s["lens"] = _table(g, lens, c["page"], pages), _ints(lens)
        s["kv"] = g.normal(c["layers"], 2, pages, *shape, dtype=c["dtype"])
        s["refs"] = _refs(s["table"], pages)
        s["table_out"], s["refs_out"] = torch.empty_like(s["table"]), torch.empty_like(s["refs"])
    else:
        lens, new = _lens(c), _new(c)
        pages = sum(-(-n // c["page"]) for n in lens) + 7
        s["table"], s["lens"] = _table(g, lens, c["page"], pages), _ints(lens)
        s["starts"] = _ints(np.concatenate([[0], np.cumsum(new)]).tolist())
        s["k"], s["v"] = g.normal(pages, *shape, dtype=c["dtype"]), g.normal(pages, *shape, dtype=c["dtype"])
        T, H, D = sum(new), c["heads"], c["dim"]
        s["T"], s["n_max"], s["l_max"] = T, max(new), max(lens)
        if c["kind"] == "rope":
            s["x"] = g.normal(T, (H + 2 * c["kv_heads"]) * D + 64, dtype=c["io"])  # the rows of a wider buffer
            s["steps"], s["mag"] = _steps(c["rot"], c["scaling"])
            s["q"] = torch.empty(T, H * D, dtype=TORCH[c["dtype"]], device="cuda")
        else:
            s["q"] = g.normal(T, H * D, dtype=c["io"], scale=1.5)
            s["slopes"] = torch.exp2(-8.0 * torch.arange(1, H + 1, device="cuda", dtype=torch.float32) / H) if c["slopes"] else None
            s["prefix"] = _ints([c["prefix"]] * c["batch"]) if c["prefix"] else None
            s["out"] = torch.empty_like(s["q"])
    return _ready(s)


def _refs(table, pages):
    return torch.bincount(table[table >= 0].long(), minlength=pages).to(torch.int32)


def _ready(s):
    if own:
        _handles(s)
    torch.cuda.synchronize()  # the inputs are made on torch's stream, the library has its own
    return s


class _Ptr:
    """A tensor as the library's calls take buffers."""

    def __init__(self, t, at=0):
        self.t, self.ptr, self.nbytes = t, t.data_ptr() + at, t.numel() * t.element_size() - at


def _buf(t):
    return None if t is None else _Ptr(t)


def _handles(s):
    """The descriptors that a program makes once for its cache, batch and options."""
    from bybylang_amd import device as dev

    dev.init(0)
    c, b = s["c"], {k: _Ptr(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
    s["dev"], s["b"] = dev, b
    if c["kind"] == "norm":
        kind = {"rms": dev.NORM_RMS, "layer": dev.NORM_LAYER}
        for at in ("post", "pre"):
            s[at] = None if c[at] == "none" else dev.Norm(kind[c[at]], 1e-5, b[at + "_w"], b[at + "_b"] if c[at] == "layer" else None)
        return
    geometry = (CODE[c["dtype"]], s["kv"].shape[2] if "kv" in s else s["k"].shape[0], c["page"], c["kv_heads"], c["dim"])
    if "kv" in s:
        s["status"] = torch.zeros(4, dtype=torch.int32, device="cuda")
        b["status"] = _Ptr(s["status"])
        caches = [dev.KvCache(_Ptr(s["kv"][i, 0]), _Ptr(s["kv"][i, 1]), *geometry) for i in range(c["layers"])]
        s["pool"] = dev.KvPool(caches, b["refs"], b["table"], s["table"].shape[1], b["lens"], s["table"].shape[0], b["status"])
        return
    s["cache"] = dev.KvCache(b["k"], b["v"], *geometry)
    s["batch"] = dev.KvBatch(b["table"], s["table"].shape[1], b["starts"], b["lens"], c["batch"], s["T"])
    if c["kind"] == "rope":
        s["rope"] = dev.Rope(dev.ROPE_HALVES if c["layout"] == "half" else dev.ROPE_PAIRS, c["rot"], b["steps"], s["mag"])
        at = [n * c["dim"] * SIZE[c["io"]] for n in (0, c["heads"], c["heads"] + c["kv_heads"])]
        s["qkv"] = [_Ptr(s["x"], a) for a in at]
    else:
        s["opts"] = dev.Attn(c["dim"] ** -0.5, c["cap"], c["window"], _buf(s["slopes"]), _buf(s["prefix"]))


# ── one pass ────────────────────────────────────────────────────────────────────────────────


def run(s):
    kind = s["c"]["kind"]
    if own:
        return {"rope": _own_rope, "attn": _own_attn, "fork": _own_fork, "compact": _own_compact, "norm": _own_norm}[kind](s)
    return {"rope": _plain_rope, "attn": _plain_attn, "fork": _plain_fork, "compact": _plain_compact, "norm": _plain_norm}[kind](s)


def _own_rope(s):
    c, b = s["c"], s["b"]
    w = s["x"].shape[1]
    q, k, v = s["qkv"]
    s["dev"].rope_append(q, w, k, w, v, w, CODE[c["io"]], c["heads"], s["rope"], s["cache"], s["batch"], b["q"], s["q"].shape[1], CODE[c["dtype"]])
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _own_attn(s):
    c, b = s["c"], s["b"]
    w = s["q"].shape[1]
    s["dev"].paged_attention(b["q"], w, CODE[c["io"]], c["heads"], s["opts"], s["cache"], s["batch"], b["out"], w, CODE[c["io"]])
    return s["out"]


def _own_fork(s):
    n, b = s["c"]["children"], s["b"]
    s["dev"].cache_fork(s["pool"], b["parents"], b["rows"], n)
    s["dev"].cache_grow(s["pool"], b["rows"], b["add"], n)
    return {"kv": s["kv"], "table": s["table"], "refs": s["refs"], "lens": s["lens"]}


def _own_compact(s):
    s["dev"].cache_compact(s["pool"], s["b"]["table_out"], s["b"]["refs_out"])
    return {"kv": s["kv"], "table": s["table_out"], "refs": s["refs_out"]}


def _own_norm(s):
    c, b = s["c"], s["b"]
    N = c["cols"]
    s["dev"].norm_block(b["x"], N, CODE[c["x"]], c["rows"], N, s["post"], b.get("gate"), 0, b["res"], N, c["scale"], b["h"], N, CODE[c["h"]],
                        s["pre"], b["y"], N, CODE[c["y"]])
    return {"h": s["h"], "y": s["y"]}


def _rows(s):
    """Each row's sequence and position."""
    t = torch.arange(s["T"], device="cuda", dtype=torch.int32)
    b = torch.searchsorted(s["starts"][1:].contiguous(), t, right=True)
    return b, s["lens"][b] - s["starts"][b + 1] + t


def _plain_rope(s):
    c = s["c"]
    H, Hk, D, T, r = c["heads"], c["kv_heads"], c["dim"], s["T"], c["rot"]
    b, pos = _rows(s)
    # the angle's whole turns fall away in the 64-bit product; what is left is a fraction of a turn
    angle = (pos.long()[:, None] * s["steps"]).float() * (math.pi / 2.0**63)
    cos, sin = (torch.cos(angle) * s["mag"])[:, None], (torch.sin(angle) * s["mag"])[:, None]
    x = s["x"][:, :(H + 2 * Hk) * D].float().view(T, H + 2 * Hk, D)
    qk = x[:, :H + Hk]
    if c["layout"] == "half":
        u, w = qk[..., :r // 2], qk[..., r // 2:r]
        turned = torch.cat([u * cos - w * sin, u * sin + w * cos], -1)
    else:
        u, w = qk[..., 0:r:2], qk[..., 1:r:2]
        turned = torch.stack([u * cos - w * sin, u * sin + w * cos], -1).flatten(-2)
    turned = torch.cat([turned, qk[..., r:]], -1)
    page, slot = s["table"][b, (pos // c["page"]).long()].long(), (pos % c["page"]).long()
    s["k"][page, :, slot] = turned[:, H:].to(s["k"].dtype)
    s["v"][page, :, slot] = x[:, H + Hk:].to(s["v"].dtype)
    return {"q": turned[:, :H].reshape(T, H * D).to(s["q"].dtype), "k": s["k"], "v": s["v"]}


def _plain_attn(s):
    c = s["c"]
    B, H, Hk, D, n, L = c["batch"], c["heads"], c["kv_heads"], c["dim"], s["n_max"], s["l_max"]
    G = H // Hk
    lens, starts = s["lens"].long(), s["starts"].long()
    new = starts[1:] - starts[:-1]
    j = torch.arange(L, device="cuda")
    there = j < lens[:, None]
    page = s["table"][:, j // c["page"]].long().clamp(min=0)
    k, v = (torch.where(there[:, :, None, None], s[x][page, :, j % c["page"]].float(), 0.0).transpose(1, 2).contiguous().view(B * Hk, L, D) for x in ("k", "v"))
    i = torch.arange(n, device="cuda")
    at = (starts[:-1, None] + i).clamp(max=s["T"] - 1)
    q = s["q"][at].float().view(B, n, Hk, G, D).permute(0, 2, 3, 1, 4).contiguous().view(B * Hk, G * n, D)
    sc = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(D ** -0.5).view(B, H, n, L)
    del q, k
    if c["cap"]:
        sc = torch.tanh(sc.div_(c["cap"])).mul_(c["cap"])
    pos = (lens - new)[:, None] + i
    back = pos[:, :, None] - j
    if s["slopes"] is not None:
        sc -= s["slopes"][:, None, None] * back[:, None].abs()
    see = back >= 0
    if c["window"]:
        see &= back < c["window"]
    if s["prefix"] is not None:
        see |= j < s["prefix"][:, None, None]
    see &= there[:, None]
    sc.masked_fill_(~see[:, None], -math.inf)
    p = torch.exp(sc - sc.amax(-1, keepdim=True).clamp(min=-3e38))
    del sc
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(B * Hk, G * n, L), v).view(B, H, n, D) / torch.where(total > 0, total, 1.0)
    b, pos = _rows(s)
    return o[b, :, (pos - (lens - new)[b]).long()].reshape(s["T"], H * D).to(s["q"].dtype)


def _plain_fork(s):
    c = s["c"]
    table, refs, lens, rows, parents = s["table"], s["refs"], s["lens"], s["rows"].long(), s["parents"].long()
    P, W, page, n = refs.numel(), table.shape[1], c["page"], c["children"]
    one = torch.ones((), dtype=torch.int32, device="cuda")

    def count(t, by):
        ids = torch.where(t >= 0, t, P).long().flatten()
        refs.copy_(torch.cat([refs, refs[:1]]).index_add(0, ids, (by * one).expand(ids.numel()))[:P])

    # fork: what the rows held is released, the parents' pages are shared
    count(table[rows], -1)
    table[rows] = table[parents]
    lens[rows] = lens[parents]
    count(table[rows], 1)
    # grow: a partly filled last page that others hold too is replaced, new pages follow it
    have, want = lens[rows], lens[rows] + s["add"]
    last = table[rows, ((have - 1).clamp(min=0) // page).long()]
    part = (have % page != 0) & (last >= 0)
    same = (last[:, None] == last) & part[:, None] & part
    before = same.tril(-1).sum(1)
    copy = part & (refs[last.clamp(min=0).long()] - before > 1)
    col = torch.arange(W, device="cuda")
    first = (have + page - 1) // page - copy.int()
    fresh = (col >= first[:, None]) & (col < ((want + page - 1) // page)[:, None])
    free = torch.argsort((refs > 0).to(torch.int32), stable=True).to(torch.int32)
    rank = fresh.flatten().cumsum(0).view(n, W) - 1
    held = table[rows]
    got = torch.where(fresh, free[rank.clamp(min=0)], held)
    gone = torch.where(copy, last, -1)
    count(gone, -1)
    count(torch.where(fresh, got, -1), 1)
    table[rows] = got
    lens[rows] = want
    src = torch.where(copy, last, 0).long()
    dst = torch.where(copy, got[torch.arange(n, device="cuda"), ((have - 1).clamp(min=0) // page).long()], 0).long()
    s["kv"][:, :, dst] = s["kv"][:, :, src]
    return {"kv": s["kv"], "table": table, "refs": refs, "lens": lens}


def _plain_compact(s):
    refs, table, P = s["refs"], s["table"], s["refs"].numel()
    live, at = refs > 0, torch.arange(P, device="cuda")
    front = at < live.sum()
    hole, mover = ~live & front, live & ~front
    src, dst = mover.nonzero().flatten(), hole.nonzero().flatten()
    remap = at.to(torch.int32).clone()
    remap[src] = dst.to(torch.int32)
    s["kv"][:, :, dst] = s["kv"][:, :, src]
    s["table_out"].copy_(torch.where(table >= 0, remap[table.clamp(min=0).long()], table))
    s["refs_out"].copy_(refs)
    s["refs_out"][dst] = refs[src]
    s["refs_out"][src] = 0
    return {"kv": s["kv"], "table": s["table_out"], "refs": s["refs_out"]}


def _plain_norm(s):
    c = s["c"]

    def norm(v, at):
        if c[at] == "none":
            return v
        if c[at] == "rms":
            return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-5) * s[at + "_w"]
        d = v - v.mean(-1, keepdim=True)
        return d * torch.rsqrt((d * d).mean(-1, keepdim=True) + 1e-5) * s[at + "_w"] + s[at + "_b"]

    x = norm(s["x"].float(), "post")
    if s["gate"] is not None:
        x = x * s["gate"]
    h = s["res"].float() * c["scale"] + x
    return {"h": h.to(s["h"].dtype), "y": norm(h, "pre").to(s["y"].dtype)}


# ── the definitions in 64 bits ──────────────────────────────────────────────────────────────


def exact(case, seed):
    """What run() returns for these inputs, from each operator's definition, sequence by sequence."""
    s, c = prepare(case, seed), case
    if c["kind"] == "norm":
        def norm(v, at):
            if c[at] == "none":
                return v
            mean = v.mean(1) if c[at] == "layer" else torch.zeros(v.shape[0], dtype=torch.float64, device="cuda")
            var = (v - mean[:, None]).pow(2).mean(1)
            out = (v - mean[:, None]) / (var + 1e-5).sqrt()[:, None] * s[at + "_w"].double()
            return out + s[at + "_b"].double() if c[at] == "layer" else out
        x = norm(s["x"].double(), "post")
        h = s["res"].double() * c["scale"] + (x if s["gate"] is None else x * s["gate"].double())
        return {"h": h, "y": norm(h, "pre")}
    if c["kind"] == "rope":
        return _exact_rope(s)
    if c["kind"] == "attn":
        return _exact_attn(s)
    return _exact_fork(s) if c["kind"] == "fork" else _exact_compact(s)


def _exact_rope(s):
    c = s["c"]
    H, Hk, D, r = c["heads"], c["kv_heads"], c["dim"], c["rot"]
    x = s["x"][:, :-64].double().cpu().numpy().reshape(s["T"], H + 2 * Hk, D)
    steps = s["steps"].cpu().numpy().view(np.uint64)
    table, t = s["table"].cpu().numpy(), 0
    k, v, q = s["k"].double(), s["v"].double(), np.empty((s["T"], H, D))
    for b, (L, n) in enumerate(zip(_lens(c), _new(c))):
        p = np.arange(L - n, L, dtype=np.uint64)
        turns = (p[:, None] * steps[None, :]).astype(np.float64) / 2.0**64
        z = np.exp(2j * np.pi * turns)[:, None, :] * s["mag"]
        rows = x[t:t + n]
        y = rows.copy()
        first, second = (slice(0, r // 2), slice(r // 2, r)) if c["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
        w = (rows[..., first] + 1j * rows[..., second]) * z
        y[..., first], y[..., second] = w.real, w.imag
        q[t:t + n] = y[:, :H]
        p = p.astype(np.int64)
        page, slot = torch.from_numpy(table[b, p // c["page"]].astype(np.int64)).cuda(), torch.from_numpy(p % c["page"]).cuda()
        k[page, :, slot] = torch.from_numpy(y[:, H:H + Hk]).cuda()
        v[page, :, slot] = torch.from_numpy(rows[:, H + Hk:]).cuda()
        t += n
    return {"q": torch.from_numpy(q.reshape(s["T"], H * D)), "k": k, "v": v}


def _exact_attn(s):
    c = s["c"]
    H, Hk, D = c["heads"], c["kv_heads"], c["dim"]
    G, t, out = H // Hk, 0, torch.zeros(s["T"], H, D, dtype=torch.float64, device="cuda")
    for b, (L, n) in enumerate(zip(_lens(c), _new(c))):
        pages = s["table"][b, :-(-L // c["page"])].long()
        key = torch.arange(L, device="cuda")
        q = s["q"][t:t + n].double().view(n, H, D)
        for h in range(Hk):
            k, v = (s[x][pages, h].reshape(-1, D)[:L].double() for x in ("k", "v"))
            for i0 in range(0, n, 1024):
                i1 = min(n, i0 + 1024)
                at = (L - n + torch.arange(i0, i1, device="cuda"))[:, None]
                seen = key <= at
                if c["window"]:
                    seen = seen & (at - key < c["window"])
                if c["prefix"]:
                    seen = seen | (key < c["prefix"])
                for g in range(h * G, (h + 1) * G):
                    z = q[i0:i1, g] @ k.T / math.sqrt(D)
                    z = c["cap"] * torch.tanh(z / c["cap"]) if c["cap"] else z
                    if c["slopes"]:
                        z = z - 2.0 ** (-8.0 * (g + 1) / H) * (at - key).abs()
                    out[t + i0:t + i1, g] = torch.softmax(z.masked_fill(~seen, -math.inf), 1) @ v
        t += n
    return out.view(s["T"], H * D)


def _exact_fork(s):
    c, kv = s["c"], s["kv"].double()
    table, refs, lens = (s[x].cpu().numpy().copy() for x in ("table", "refs", "lens"))
    for i in range(c["children"]):
        a, r = i % c["parents"], c["parents"] + i
        table[r], lens[r] = table[a], lens[a]
        for p in table[r][table[r] >= 0]:
            refs[p] += 1
    for r in range(c["parents"], c["parents"] + c["children"]):
        at, end = int(lens[r]), int(lens[r]) + c["add"]
        if at % c["page"] and refs[table[r, at // c["page"]]] > 1:
            old = int(table[r, at // c["page"]])
            new = int(np.flatnonzero(refs == 0)[0])
            kv[:, :, new] = kv[:, :, old]
            refs[old] -= 1
            refs[new], table[r, at // c["page"]] = 1, new
        for col in range(-(-at // c["page"]), -(-end // c["page"])):
            table[r, col] = np.flatnonzero(refs == 0)[0]
            refs[table[r, col]] = 1
        lens[r] = end
    return {"kv": kv, "table": table, "refs": refs, "lens": lens}


def _exact_compact(s):
    kv, refs, table = s["kv"].double(), s["refs"].cpu().numpy().copy(), s["table"].cpu().numpy().copy()
    live = int((refs > 0).sum())
    moved = {}
    for src in [p for p in range(live, len(refs)) if refs[p] > 0]:
        dst = int(np.flatnonzero(refs[:live] == 0)[0])
        refs[dst], refs[src] = refs[src], 0
        moved[src] = dst
    if moved:
        kv[:, :, torch.tensor(list(moved.values())).cuda()] = kv[:, :, torch.tensor(list(moved.keys())).cuda()]
    table = np.vectorize(lambda p: moved.get(p, p), otypes=[np.int32])(table)
    return {"kv": kv, "table": table, "refs": refs}
