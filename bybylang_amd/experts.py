"""A block of experts on the session API: the residual's addition and an RMS norm into 8 bits, router logits, routing, the
experts' products with silu(gate) * up between them, and each token's weighted sum. Every weight is a matrix in 4 bits (FP4-KM
with E8M0 scales). `python -m bybylang_amd.paged_decoder --experts 64` runs it after each attention block.
"""
from __future__ import annotations

import numpy as np

from . import _abi, device as dev, gpubackend as g, synth
from .gpubackend import gbHip


def random_matrix(rng, rows: int, width: int) -> g.SessionHandle:
    """`rows` rows of `width` values in 4 bits, of the size that keeps a normed row's products near 1."""
    codes = synth.fp4km_pack(rng.integers(0, 16, (rows, width), dtype=np.uint8))
    scale = 127 + int(np.round(np.log2(0.4 / np.sqrt(width))))
    blob = np.concatenate([codes.reshape(-1), np.full(rows * width // 32, scale, np.uint8)])
    return g.sessionUploadBytes(gbHip, blob)


class ExpertsBlock:
    """`experts` experts of `inner` values over rows of `width`, `top_k` per token, for up to `max_rows` rows a call.

    router [experts, width], up [experts, 2 inner, width] (gates, then ups, of each expert) and down [experts, width, inner]:
    handles of matrices in 4 bits; rows are 8-bit ones throughout, the router's too. norm: gammas of the RMS norm before the block; bias: fp32 [experts] added to the scores for the choice
    only, or None. exact: BYHIP_MOE_EXACT of the experts' products."""

    def __init__(self, router, up, down, norm, width: int, inner: int, experts: int, top_k: int, max_rows: int, eps: float = 1e-5,
                 score: int = _abi.MOE_SOFTMAX, bias=None, groups: int = 1, top_groups: int = 1, group_by: int = 1, renorm: bool = True,
                 scale: float = 1.0, exact: bool = False):
        self.weights, self.width, self.inner, self.experts, self.top_k = (router, up, down), width, inner, experts, top_k
        self.norm = dev.Norm(_abi.NORM_RMS, eps, g.sessionUpload(gbHip, norm))
        self.router = dev.MoeRouter(score, None if bias is None else g.sessionUpload(gbHip, bias), groups, top_groups, group_by, renorm, scale)
        self.exact = _abi.MOE_EXACT * exact
        self.max_rows, rows = max_rows, max_rows * top_k
        # A plan of fewer tokens may have shorter units, and more of them.
        self.plan_buffer = g.sessionAllocBytes(gbHip, max(dev.moe_plan_bytes(t, top_k, experts) for t in range(1, max_rows + 1)))
        self.xq = g.sessionAllocBytes(gbHip, dev.mx_bytes(max_rows, width, _abi.MXFP8_KM))
        self.mid = g.sessionAllocBytes(gbHip, dev.mx_bytes(rows, inner, _abi.MXFP8_KM))
        self.logits, self.ids, self.shares = (g.sessionAllocScratch(gbHip, n) for n in (max_rows * experts, rows, rows))
        self.rows = g.sessionAllocScratch(gbHip, rows * width)

    def encode(self, x: g.SessionHandle, T: int, h: g.SessionHandle, out: g.SessionHandle) -> bool:
        """h += x, out = the block of h (T rows; out may be x). False where an operator does not take the sizes."""
        router, up, down = self.weights
        D, F, mx8 = self.width, self.inner, _abi.MXFP8_KM
        plan = dev.MoePlan(self.plan_buffer, T, self.top_k, self.experts)
        ok = g.sessionNormBlockMx(gbHip, x, T, D, None, None, h, 1.0, h, self.norm, self.xq, mx8)
        ok &= g.sessionMxMatmul(gbHip, self.xq, mx8, router, T, D, self.experts, self.logits)
        ok &= g.sessionMoeRoute(gbHip, self.logits, self.router, plan, self.ids, self.shares)
        ok &= g.sessionMoeMatmul(gbHip, self.xq, mx8, up, plan, D, F, _abi.MOE_GATHER | _abi.MOE_SWIGLU | self.exact, self.mid, mx8)
        ok &= g.sessionMoeMatmul(gbHip, self.mid, mx8, down, plan, F, D, _abi.MOE_SCATTER, self.rows)
        return ok and g.sessionMoeCombine(gbHip, self.rows, D, plan, self.ids, self.shares, None, out)
