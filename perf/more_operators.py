"""Performance cases of a block of experts on microscaled weights: what a serving program calls between the
attention of a decoder layer and the next one's.

Kinds
  norm   norm_block into 8 bits: the residual's addition and an RMS norm whose rows come out as e4m3 values with
         one power-of-two scale per 32.
  quant  mx_quantize and mx_matmul: rows in 32 or 16 bits to 8 or 4 bits with scales, and their product with a
         matrix in 4 bits.
  route  moe_route: scores of the experts, the best of them per token with their weights, and the plan that
         orders the tokens by expert.
  up     moe_matmul of the tokens with their experts' gate and up matrices, silu(gate) * up in the epilogue.
  down   moe_matmul of those rows with their experts' down matrices, and moe_combine of each token's rows.

Microscaled rows of K values, M of them, are M K (8 bits) or M K / 2 bytes (4 bits), then M K / 32 scale bytes
(2^(byte - 127)). Within 32 values, the order in memory is 0, 16, 1, 17, .., 15, 31; in 4 bits the first of two
is the low nibble. A scale is the least power of two with which the largest of its 32 values is in the format's
range (448, or 6); values are rounded to the nearest, ties to even.
"""
import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "mx8": 33 / 32, "mx4": 17 / 32}
CODE = {"f32": 0, "f16": 1, "bf16": 2, "mx4": 3, "mx8": 4}


def listed():
    return [
        # the residual stream of one decode step of 32 sequences: latency
        {"name": "norm_decode", "kind": "norm", "rows": 32, "cols": 4096, "x": "f32", "h": "f32"},
        # the residual stream of a prompt of no round length
        {"name": "norm_prompt", "kind": "norm", "rows": 4099, "cols": 5120, "x": "bf16", "h": "f32"},
        # a decode step's rows, quantised to 8 bits, times one projection
        {"name": "quant_decode", "kind": "quant", "rows": 16, "K": 4096, "N": 14336, "x": "f32", "fmt": "mx8", "y": "f32"},
        # a prompt's rows, quantised to 4 bits, times one projection
        {"name": "quant_prompt", "kind": "quant", "rows": 2047, "K": 4096, "N": 4096, "x": "bf16", "fmt": "mx4", "y": "bf16"},
        # one decode step of 32 sequences, softmax scores of 128 experts, 8 each
        {"name": "route_decode", "kind": "route", "rows": 32, "experts": 128, "top": 8, "logits": "f32", "score": "softmax", "bias": False, "groups": 1, "top_groups": 1, "renorm": True},
        # prompts, sigmoid scores with a bias for balance, 4 of 8 groups of 256 experts
        {"name": "route_prompt", "kind": "route", "rows": 8191, "experts": 256, "top": 8, "logits": "f32", "score": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "renorm": True},
        # one token: latency
        {"name": "up_one", "kind": "up", "rows": 1, "experts": 64, "top": 8, "K": 2048, "N": 1024, "x": "mx8", "y": "mx8"},
        # one decode step of 48 sequences: nearly every expert's matrices are read for a few rows each
        {"name": "up_decode", "kind": "up", "rows": 48, "experts": 128, "top": 8, "K": 2048, "N": 768, "x": "mx8", "y": "mx8"},
        # a chunk of a prompt over a few large experts, activations in 4 bits
        {"name": "up_chunk", "kind": "up", "rows": 509, "experts": 16, "top": 2, "K": 4096, "N": 2048, "x": "mx4", "y": "f16"},
        # prompts: hundreds of rows per expert
        {"name": "up_prompt", "kind": "up", "rows": 4096, "experts": 64, "top": 6, "K": 2048, "N": 1408, "x": "mx8", "y": "mx8"},
        # the down half of the decode step, into an fp32 stream
        {"name": "down_decode", "kind": "down", "rows": 48, "experts": 128, "top": 8, "K": 768, "N": 2048, "x": "mx8", "mid": "f32", "y": "f32"},
        # the down half of the prompts
        {"name": "down_prompt", "kind": "down", "rows": 4096, "experts": 64, "top": 6, "K": 1408, "N": 2048, "x": "mx8", "mid": "bf16", "y": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the listed ones' ranges, at most the largest one's work."""
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= 3.5e8 and w["flops"] <= 2.8e11:
            return case


def _draw(rng):
    kind = rng.choice(["norm", "quant", "route", "up", "up", "down", "down"])
    if kind == "norm":
        x = rng.choice(["f32", "f16", "bf16"])
        return {"kind": kind, "rows": _log(rng, 1, 8192), "cols": 32 * _log(rng, 8, 512), "x": x, "h": rng.choice(["f32", x])}
    if kind == "quant":
        K = 32 * _log(rng, 16, 448)
        fmt = rng.choice(["mx8", "mx4"])
        return {"kind": kind, "rows": _log(rng, 1, 4096), "K": K if rng.random() < 0.4 else -(-K // 128) * 128, "N": _log(rng, 100, 14336), "x": rng.choice(["f32", "f16", "bf16"]),
                "fmt": fmt, "y": rng.choice(["f32", "f16", "bf16"])}
    if kind == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * _log(rng, 8 // groups + 1, 512 // groups)
        top_groups = rng.randint(1, groups)
        return {"kind": kind, "rows": _log(rng, 1, 16384), "experts": experts, "top": min(experts // groups * top_groups, rng.choice([1, 2, 4, 6, 8, 8, 10])),
                "logits": rng.choice(["f32", "f32", "bf16", "f16"]), "score": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups,
                "renorm": rng.random() < 0.7}
    experts = _log(rng, 4, 160)
    c = {"kind": kind, "rows": _log(rng, 1, 8192), "experts": experts, "top": min(experts, rng.choice([1, 2, 4, 6, 8, 8])), "K": 32 * _log(rng, 16, 128), "N": 32 * _log(rng, 12, 128)}
    if kind == "up":
        return {**c, "x": rng.choice(["mx8", "mx8", "mx4"]), "y": rng.choice(["mx8", "mx8", "f16", "bf16"])}
    y = rng.choice(["f32", "bf16", "f16"])
    return {**c, "x": rng.choice(["mx8", "mx8", "mx4"]), "mid": y, "y": y}


def _popularity(c):
    """Experts are not asked for alike: their logits' offsets."""
    return 0.6 * torch.randn(c["experts"], generator=torch.Generator().manual_seed(c["experts"]))


def _chosen(c, seed):
    """Each token's experts [rows, top], on the host."""
    g = torch.Generator().manual_seed(int(seed) * 31 + 5)
    return torch.topk(torch.randn(c["rows"], c["experts"], generator=g) + _popularity(c), c["top"], dim=1).indices.to(torch.int32)


def work(c):
    k, T = c["kind"], c["rows"]
    if k == "norm":
        n = T * c["cols"]
        return {"bytes": n * (SIZE[c["x"]] + 2 * SIZE[c["h"]] + SIZE["mx8"]) + 4 * c["cols"], "flops": 8 * n}
    if k == "quant":
        return {"bytes": T * c["K"] * SIZE[c["x"]] + c["N"] * c["K"] * SIZE["mx4"] + T * c["N"] * SIZE[c["y"]], "flops": 2 * T * c["K"] * c["N"]}
    A = T * c["top"]
    if k == "route":
        return {"bytes": T * c["experts"] * SIZE[c["logits"]] + 12 * A + 4 * c["experts"], "flops": 6 * T * c["experts"]}
    used = int(torch.unique(_chosen(c, 0)).numel())
    if k == "up":
        return {"bytes": T * c["K"] * SIZE[c["x"]] + used * 2 * c["N"] * c["K"] * SIZE["mx4"] + A * c["N"] * SIZE[c["y"]], "flops": 4 * A * c["K"] * c["N"]}
    return {"bytes": A * c["K"] * SIZE[c["x"]] + used * c["N"] * c["K"] * SIZE["mx4"] + 2 * T * c["N"] * SIZE[c["y"]], "flops": 2 * A * c["K"] * c["N"]}


# ── microscaled rows in plain torch ─────────────────────────────────────────────────────────


def _two_to(e):
    """2^(byte - 127) of int32 scale bytes (0 stands for the least, 2^-127)."""
    return torch.where(e > 0, e << 23, 1 << 22).view(torch.float32)


def _quantize(v, fmt):
    """fp32 [R, K] -> (codes, scale bytes [R, K / 32]): e4m3 values [R, K], or nibbles [R, K / 2]."""
    R, K = v.shape
    v = v.view(R, K // 32, 32)
    bits = v.abs().amax(-1).view(torch.int32)
    # the largest value is m 2^x with 1 <= m < 2; it is in range where the scale is 2^(x - 8) and m <= 1.75 (448), 2^(x - 2) and m <= 1.5 (6)
    step, most = (8, 0x600000) if fmt == "mx8" else (2, 0x400000)
    e = ((bits >> 23) - step + ((bits & 0x7FFFFF) > most).int()).clamp(min=0)
    v = v * (1.0 / _two_to(e))[..., None]
    if fmt == "mx8":
        codes = v.view(R, K // 32, 2, 16).transpose(2, 3).reshape(R, K).to(torch.float8_e4m3fn)
    else:
        a = v.abs()
        n = (a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5) + 8 * torch.signbit(v).byte()
        codes = (n[..., :16] | (n[..., 16:] << 4)).view(R, K // 2)
    return codes, e.to(torch.uint8)


def _values(codes, scales, fmt):
    """(codes, scale bytes) -> fp32 [R, K]."""
    R, groups = scales.shape
    if fmt == "mx8":
        v = codes.view(torch.float8_e4m3fn).float().view(R, groups, 16, 2).transpose(2, 3).reshape(R, groups, 32)
    else:
        b = codes.view(R, groups, 16).int()
        n = torch.cat([b & 15, b >> 4], -1)
        m = n & 7
        v = torch.where(m < 2, 0.5 * m, (1 + 0.5 * (m & 1)) * (1 << (m >> 1)) * 0.5)
        v = torch.where(n > 7, -v, v)
    return (v * _two_to(scales.int())[..., None]).view(R, groups * 32)


def _row_bytes(K, fmt):
    return K if fmt == "mx8" else K // 2


def _halves(buf, R, K, fmt):
    """A buffer of microscaled rows -> its codes [R, ..] and scale bytes [R, K / 32]."""
    n = R * _row_bytes(K, fmt)
    return buf[:n].view(R, -1), buf[n:n + R * K // 32].view(R, K // 32)


def _answer(codes, scales):
    """Rows in 8 bits as what they stand for: the values, and the powers of two they are multiplied by."""
    return {"values": codes.view(torch.float8_e4m3fn), "scales": scales.view(torch.float8_e8m0fnu)}


# ── inputs ──────────────────────────────────────────────────────────────────────────────────


class Gen:
    """Seeded inputs on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 29)

    def normal(self, *shape, scale=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda").mul_(scale)

    def rows(self, M, K):
        """Activations: some columns are larger than others."""
        return self.normal(M, K) * torch.exp(0.7 * self.normal(K))

    def mx(self, v, fmt):
        return torch.cat([t.view(torch.uint8).flatten() for t in _quantize(v, fmt)])

    def weights(self, count, R, K):
        """`count` matrices in 4 bits: the nibbles of all of them, then their scales."""
        parts = [_quantize(self.normal(R, K, scale=K ** -0.5), "mx4") for _ in range(count)]
        return torch.cat([p[0].flatten() for p in parts] + [p[1].flatten() for p in parts])


def prepare(case, seed):
    """Inputs, weights, the plan and the buffers as a serving program holds them before the call."""
    c, g = case, Gen(seed)
    s, T = {"c": c}, c["rows"]
    if c["kind"] == "norm":
        N = c["cols"]
        s["x"], s["res"] = g.rows(T, N).to(TORCH[c["x"]]), g.normal(T, N, scale=2.0).to(TORCH[c["h"]])
        s["w"] = 1 + g.normal(N, scale=0.2)
        s["h"], s["y"] = torch.empty(T, N, dtype=TORCH[c["h"]], device="cuda"), torch.empty(T * N // 32 * 33, dtype=torch.uint8, device="cuda")
    elif c["kind"] == "quant":
        s["x"], s["w"] = g.rows(T, c["K"]).to(TORCH[c["x"]]), g.weights(1, c["N"], c["K"])
        s["xq"] = torch.empty(T * (_row_bytes(c["K"], c["fmt"]) + c["K"] // 32), dtype=torch.uint8, device="cuda")
        s["y"] = torch.empty(T, c["N"], dtype=TORCH[c["y"]], device="cuda")
    elif c["kind"] == "route":
        E, k = c["experts"], c["top"]
        s["logits"] = (1.3 * g.normal(T, E) + _popularity(c).cuda()).to(TORCH[c["logits"]])
        s["bias"] = 0.1 * g.normal(E) if c["bias"] else None
        s["ids"], s["weights"] = torch.empty(T, k, dtype=torch.int32, device="cuda"), torch.empty(T, k, device="cuda")
    else:
        E, K, A = c["experts"], c["K"], T * c["top"]
        ids = _chosen(c, seed)
        count = torch.bincount(ids.flatten(), minlength=E)
        s["most"], used = int(count.max()), torch.nonzero(count).flatten()
        s["ids"], s["used"] = ids.cuda(), used.cuda()
        s["slot"] = torch.zeros(E, dtype=torch.long).index_copy_(0, used, torch.arange(used.numel())).cuda()
        s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.long), count.cumsum(0)]).cuda()
        s["order"] = torch.sort(ids.flatten(), stable=True).indices.cuda()
        R = 2 * c["N"] if c["kind"] == "up" else c["N"]
        s["w"] = g.weights(E, R, K)
        if c["kind"] == "up":
            s["x"] = g.mx(g.rows(T, K), c["x"])
            s["y"] = torch.empty(A * c["N"] // 32 * 33, dtype=torch.uint8, device="cuda") if c["y"] == "mx8" else torch.empty(A, c["N"], dtype=TORCH[c["y"]], device="cuda")
        else:
            s["x"] = g.mx(g.rows(A, K), c["x"])
            s["weights"] = torch.softmax(g.normal(T, c["top"]), 1)
            s["res"] = g.normal(T, c["N"], scale=2.0).to(TORCH[c["y"]])
            s["mid"], s["y"] = torch.empty(A, c["N"], dtype=TORCH[c["mid"]], device="cuda"), torch.empty(T, c["N"], dtype=TORCH[c["y"]], device="cuda")
    if own:
        _handles(s)
    torch.cuda.synchronize()  # the inputs are made on torch's stream, the library has its own
    return s


class _Ptr:
    """A tensor as the library's calls take buffers."""

    def __init__(self, t):
        self.t, self.ptr, self.nbytes = t, t.data_ptr(), t.numel() * t.element_size()


def _handles(s):
    """The descriptors that a program makes once, and the plan that its routing left."""
    from bybylang_amd import device as dev

    dev.init(0)
    c = s["c"]
    s["dev"], s["b"] = dev, {k: _Ptr(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
    b = s["b"]
    if c["kind"] == "norm":
        s["pre"] = dev.Norm(dev.NORM_RMS, 1e-5, b["w"])
        s["out"] = {"h": s["h"], **_answer(*_halves(s["y"], c["rows"], c["cols"], "mx8"))}
    if c["kind"] in ("route", "up", "down"):
        s["plan_buf"] = torch.empty(dev.moe_plan_bytes(c["rows"], c["top"], c["experts"]), dtype=torch.uint8, device="cuda")
        s["plan"] = dev.MoePlan(_Ptr(s["plan_buf"]), c["rows"], c["top"], c["experts"])
    if c["kind"] == "route":
        s["router"] = dev.MoeRouter(dev.MOE_SOFTMAX if c["score"] == "softmax" else dev.MOE_SIGMOID, b.get("bias"), c["groups"], c["top_groups"],
                                    2 if c["bias"] else 1, c["renorm"], 2.5 if c["score"] == "sigmoid" else 1.0)
        ints, E = s["plan_buf"].view(torch.int32), c["experts"]
        s["out"] = {"ids": s["ids"], "weights": s["weights"], "offsets": ints[:E + 1], "order": ints[E + 1:E + 1 + s["ids"].numel()]}
    if c["kind"] in ("up", "down"):
        torch.cuda.synchronize()  # torch's work on memory that the plan's buffer was given is over before the library writes there
        dev.moe_plan(b["ids"], s["plan"])
        dev.synchronize()
        s["out"] = _answer(*_halves(s["y"], c["rows"] * c["top"], c["N"], "mx8")) if c["y"] == "mx8" else {"y": s["y"]}


# ── one pass ────────────────────────────────────────────────────────────────────────────────


def run(s):
    kind = s["c"]["kind"]
    if own:
        return {"norm": _own_norm, "quant": _own_quant, "route": _own_route, "up": _own_up, "down": _own_down}[kind](s)
    return {"norm": _plain_norm, "quant": _plain_quant, "route": _plain_route, "up": _plain_up, "down": _plain_down}[kind](s)


def _own_norm(s):
    c, b, N = s["c"], s["b"], s["c"]["cols"]
    s["dev"].norm_block(b["x"], N, CODE[c["x"]], c["rows"], N, None, None, 0, b["res"], N, 1.0, b["h"], N, CODE[c["h"]], s["pre"], b["y"], N, CODE["mx8"])
    return s["out"]


def _own_quant(s):
    c, b = s["c"], s["b"]
    s["dev"].mx_quantize(b["x"], c["K"], CODE[c["x"]], c["rows"], c["K"], b["xq"], CODE[c["fmt"]])
    s["dev"].mx_matmul(b["xq"], CODE[c["fmt"]], b["w"], c["rows"], c["K"], c["N"], 0, b["y"], c["N"], CODE[c["y"]])
    return s["y"]


def _own_route(s):
    c, b = s["c"], s["b"]
    s["dev"].moe_route(b["logits"], c["experts"], CODE[c["logits"]], s["router"], s["plan"], b["ids"], b["weights"])
    return s["out"]


def _own_up(s):
    c, b, dev = s["c"], s["b"], s["dev"]
    dev.moe_matmul(b["x"], CODE[c["x"]], b["w"], s["plan"], c["K"], c["N"], dev.MOE_GATHER | dev.MOE_SWIGLU, b["y"], c["N"], CODE[c["y"]])
    return s["out"]


def _own_down(s):
    c, b, dev = s["c"], s["b"], s["dev"]
    dev.moe_matmul(b["x"], CODE[c["x"]], b["w"], s["plan"], c["K"], c["N"], dev.MOE_SCATTER, b["mid"], c["N"], CODE[c["mid"]])
    dev.moe_combine(b["mid"], c["N"], CODE[c["mid"]], c["N"], s["plan"], b["ids"], b["weights"], b["res"], c["N"], CODE[c["y"]], b["y"], c["N"], CODE[c["y"]])
    return s["y"]


def _plain_norm(s):
    h = s["res"].float() + s["x"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-5) * s["w"]
    return {"h": h.to(s["h"].dtype), **_answer(*_quantize(y, "mx8"))}


def _plain_quant(s):
    c = s["c"]
    x = _values(*_quantize(s["x"].float(), c["fmt"]), c["fmt"])
    w = _values(*_halves(s["w"], c["N"], c["K"], "mx4"), "mx4")
    return (x @ w.t()).to(s["y"].dtype)


def _plain_route(s):
    c, x = s["c"], s["logits"].double()  # two experts' scores may lie next to each other
    T, E, k, G = c["rows"], c["experts"], c["top"], c["groups"]
    if c["score"] == "softmax":
        x = torch.exp(x - x.amax(-1, keepdim=True))
        score = x / x.sum(-1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-x))
    key = score if s["bias"] is None else score + s["bias"].double()
    if G > 1:
        group = torch.sort(key.view(T, G, E // G), dim=-1, descending=True).values[..., :2 if c["bias"] else 1].sum(-1)
        best = torch.sort(group, dim=-1, descending=True, stable=True).indices[:, :c["top_groups"]]
        inside = torch.zeros(T, G, dtype=torch.bool, device="cuda").scatter_(1, best, True)
        key = torch.where(inside.repeat_interleave(E // G, dim=1), key, -math.inf)
    ids = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :k]
    w = score.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    if c["score"] == "sigmoid":
        w = w * 2.5
    flat = ids.flatten()
    count = (flat[:, None] == torch.arange(E, device="cuda")).sum(0)
    offsets = torch.cat([count[:1] * 0, count.cumsum(0)])
    return {"ids": ids.int(), "weights": w.float(), "offsets": offsets.int(), "order": torch.sort(flat, stable=True).indices.int()}


def _plain_product(s, x, packed):
    """Rows of the experts' products in the plan's order: fp32 [rows * top, matrix rows]."""
    c = s["c"]
    R = 2 * c["N"] if c["kind"] == "up" else c["N"]
    E, K, A = c["experts"], c["K"], c["rows"] * c["top"]
    at = s["offsets"][s["used"]][:, None] + torch.arange(s["most"], device="cuda")
    row = at.clamp(max=A - 1)
    rows = x[row] if packed else x[s["order"][row] // c["top"]]
    codes, scales = _halves(s["w"], E, R * K, "mx4")
    w = _values(codes[s["used"]].view(-1, K // 2), scales[s["used"]].view(-1, K // 32), "mx4").view(-1, R, K)
    y = torch.bmm(rows, w.transpose(1, 2).contiguous())
    t = torch.arange(A, device="cuda")
    e = torch.searchsorted(s["offsets"], t, right=True) - 1
    return y[s["slot"][e], t - s["offsets"][e]]


def _plain_up(s):
    c, N = s["c"], s["c"]["N"]
    v = _plain_product(s, _values(*_halves(s["x"], c["rows"], c["K"], c["x"]), c["x"]), False)
    y = v[:, :N] / (1 + torch.exp(-v[:, :N])) * v[:, N:]
    return _answer(*_quantize(y, "mx8")) if c["y"] == "mx8" else {"y": y.to(TORCH[c["y"]])}


def _plain_down(s):
    c = s["c"]
    T, k = c["rows"], c["top"]
    v = _plain_product(s, _values(*_halves(s["x"], T * k, c["K"], c["x"]), c["x"]), True)
    mid = torch.empty_like(v)
    mid[s["order"]] = v
    return (s["res"].float() + (mid.view(T, k, -1) * s["weights"][..., None]).sum(1)).to(s["y"].dtype)


# ── the definitions in 64 bits ──────────────────────────────────────────────────────────────


def _mx_exact(y, fmt):
    """float64 [R, K] -> (values in memory order, powers of two, the rows they stand for)."""
    R, K = y.shape
    v = y.view(R, -1, 32)
    most, digits, least = (448.0, 3, -6) if fmt == "mx8" else (6.0, 1, 0)
    power = torch.exp2(torch.ceil(torch.log2(v.abs().amax(-1, keepdim=True) / most)).clamp(min=-127))
    power = torch.where(v.abs().amax(-1, keepdim=True) > most * power, 2 * power, power)
    z = v / power
    grid = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** least))) - digits)
    z = torch.round(z / grid) * grid
    return z.view(R, -1, 2, 16).transpose(2, 3).reshape(R, K), power[..., 0], (z * power).view(R, K)


def _rows_exact(buf, R, K, fmt):
    """The float64 rows of a microscaled buffer, from the formats' bits."""
    codes, scales = _halves(buf, R, K, fmt)
    codes = codes.long()
    if fmt == "mx4":
        codes = torch.stack([codes & 15, codes >> 4], -1)
        exp_bits, man, bias = (codes >> 1) & 3, codes & 1, 1
        unit, sign = 2, codes >> 3
    else:
        exp_bits, man, bias = (codes >> 3) & 15, codes & 7, 7
        unit, sign = 8, codes >> 7
    v = torch.where(exp_bits > 0, (man.double() / unit + 1) * torch.exp2((exp_bits - bias).double()), man.double() / unit * 2.0 ** (1 - bias))
    v = v * (1 - 2 * sign)
    v = v.view(R, K // 32, 16, 2).permute(0, 1, 3, 2).reshape(R, K // 32, 32)
    return (v * torch.exp2(scales.double() - 127)[..., None]).view(R, K)


def exact(case, seed):
    """What run() returns for these inputs, from each operator's definition, expert by expert."""
    s, c = prepare(case, seed), case
    T = c["rows"]
    if c["kind"] == "norm":
        h = s["res"].double() + s["x"].double()
        values, power, _ = _mx_exact(h / (h.pow(2).mean(1) + 1e-5).sqrt()[:, None] * s["w"].double(), "mx8")
        return {"h": h, "values": values, "scales": power}
    if c["kind"] == "quant":
        return _mx_exact(s["x"].double(), c["fmt"])[2] @ _rows_exact(s["w"], c["N"], c["K"], "mx4").T
    if c["kind"] == "route":
        return _exact_route(s)
    E, K, k, N = c["experts"], c["K"], c["top"], c["N"]
    R = 2 * N if c["kind"] == "up" else N
    x = _rows_exact(s["x"], T if c["kind"] == "up" else T * k, K, c["x"])
    out = torch.empty(T * k, N, dtype=torch.float64, device="cuda")
    ids, at = s["ids"].flatten(), 0
    nibbles, scales = s["w"][:E * R * K // 2].view(E, -1), s["w"][E * R * K // 2:].view(E, -1)
    for e in range(E):
        who = torch.nonzero(ids == e).flatten()
        n = who.numel()
        if not n:
            continue
        w = _rows_exact(torch.cat([nibbles[e], scales[e]]), R, K, "mx4")
        if c["kind"] == "up":
            v = x[who // k] @ w.T
            out[at:at + n] = v[:, :N] * torch.sigmoid(v[:, :N]) * v[:, N:]
        else:
            out[who] = x[at:at + n] @ w.T
        at += n
    if c["kind"] == "up":
        if c["y"] != "mx8":
            return {"y": out}
        values, power, _ = _mx_exact(out, "mx8")
        return {"values": values, "scales": power}
    return s["res"].double() + (out.view(T, k, N) * s["weights"].double()[..., None]).sum(1)


def _exact_route(s):
    c = s["c"]
    T, E, G = c["rows"], c["experts"], c["groups"]
    x = s["logits"].double().cpu()
    score = torch.softmax(x, 1) if c["score"] == "softmax" else torch.sigmoid(x)
    key = score + (s["bias"].double().cpu() if c["bias"] else 0)
    ids = torch.empty(T, c["top"], dtype=torch.int64)
    for t in range(T):
        row = key[t].tolist()
        size = E // G
        if G > 1:
            worth = [sum(sorted(row[g * size:(g + 1) * size])[-2 if c["bias"] else -1:]) for g in range(G)]
            kept = sorted(range(G), key=lambda g: (-worth[g], g))[:c["top_groups"]]
            pool = [e for g in kept for e in range(g * size, (g + 1) * size)]
        else:
            pool = range(E)
        ids[t] = torch.tensor(sorted(pool, key=lambda e: (-row[e], e))[:c["top"]])
    w = torch.gather(score, 1, ids)
    w = w / w.sum(1, keepdim=True) if c["renorm"] else w
    count = torch.bincount(ids.flatten(), minlength=E)
    by = sorted(range(ids.numel()), key=ids.flatten().tolist().__getitem__)
    return {"ids": ids.int(), "weights": w * (2.5 if c["score"] == "sigmoid" else 1.0), "offsets": torch.cat([torch.zeros(1, dtype=torch.long), count.cumsum(0)]).int(),
            "order": torch.tensor(by, dtype=torch.int32)}
