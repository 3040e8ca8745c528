"""Attention blocks over a paged cache, on the session API: the residual stream, Q4 projections, rotary
positions, and a cache whose sequences grow, fork, end and are compacted.

`python -m bybylang_amd.paged_decoder` runs it: ragged prompts, beams that share their prompt's pages,
recorded decode steps. A step reads its lengths from the device and grows them itself, so that one
recording, replayed, is every further step. A slot that finds no room (no free page, or `max_len` reached) keeps
its tokens and brings none: its rows of the output hold the stream without attention, and `granted` says so.
"""
from __future__ import annotations

import argparse
import time

import numpy as np

from . import _abi, device as dev, gpubackend as g
from .gpubackend import gbHip


def random_weights(rng, K: int, N: int, group: int = 32) -> g.ResidentWeightHandle:
    groups = K // group
    scales = rng.uniform(0.5, 1.5, N * groups).astype(np.float32) * np.float32(0.2 / np.sqrt(K))
    zeros = (-7.5 * scales).astype(np.float32)
    return g.residentUploadQ4(gbHip, rng.integers(0, 256, N * K // 2, dtype=np.uint8), scales, zeros, K, N, group, groups)


def _ints(values) -> g.SessionHandle:
    return g.sessionUploadBytes(gbHip, np.asarray(values, np.int32).view(np.uint8).reshape(-1))


class PagedDecoder:
    """`layers` attention blocks of `heads` query and `kv_heads` key heads of `head_dim` values over a
    residual stream of `width` values, for up to `slots` sequences of `max_len` tokens and `max_rows` rows a call.

    layers: a list of (wq, wk, wv, wo) resident Q4 weights; norms: gammas of the RMS norm before each layer and
    after the last one."""

    def __init__(self, layers, norms, width: int, heads: int, kv_heads: int, head_dim: int, slots: int, max_len: int,
                 max_rows: int, pages: int, page_size: int = 32, cache_dtype: int = _abi.F16, eps: float = 1e-5,
                 rope_base: float = 10000.0, window: int = 0, softcap: float = 0.0):
        self.layers, self.width, self.heads, self.slots, self.max_rows = layers, width, heads, slots, max_rows
        self.stride = -(-max_len // page_size)
        scratch = lambda n: g.sessionAllocScratch(gbHip, n)  # noqa: E731
        halves = pages * kv_heads * page_size * head_dim
        self.caches = [dev.KvCache(scratch(-(-halves // 2)), scratch(-(-halves // 2)), cache_dtype, pages, page_size, kv_heads, head_dim)
                       for _ in layers]
        self.table = _ints(np.full(slots * self.stride, -1))
        self.lens, self.refs, self.status = _ints([0] * slots), _ints([0] * pages), _ints([0] * 4)
        self.room = _ints([0] * slots)
        self.pool = dev.KvPool(self.caches, self.refs, self.table, self.stride, self.lens, slots, self.status, self.room)
        self.starts, self.add, self.all_rows = _ints([0] * (slots + 1)), _ints([0] * slots), _ints(range(slots))
        self.some, self.others = _ints([0] * slots), _ints([0] * slots)
        steps, magnitude = dev.rope_steps(head_dim, rope_base)
        self.rope = dev.Rope(_abi.ROPE_HALVES, head_dim, g.sessionUploadBytes(gbHip, steps.view(np.uint8)), magnitude)
        self.attn = dev.Attn(head_dim ** -0.5, softcap, window)
        self.norms = [dev.Norm(_abi.NORM_RMS, eps, g.sessionUpload(gbHip, n)) for n in norms]
        q, kv = heads * head_dim, kv_heads * head_dim
        self.x, self.h, self.y, self.o = (scratch(max_rows * width) for _ in range(4))
        self.q, self.q_rot, self.a = (scratch(max_rows * q) for _ in range(3))
        self.k, self.v = (scratch(max_rows * kv) for _ in range(2))

    def _set(self, handle: g.SessionHandle, values) -> None:
        a = np.ascontiguousarray(values)
        _abi.check(_abi.load().byhip_upload(handle.ptr, 0, a.ctypes.data, a.nbytes), "byhip_upload")

    def set_rows(self, counts) -> None:
        """How many new rows each slot brings to the calls that follow (0: none)."""
        assert len(counts) == self.slots and sum(counts) <= self.max_rows
        self.rows = int(sum(counts))
        self._set(self.starts, np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        self._set(self.add, np.asarray(counts, np.int32))
        self.batch = dev.KvBatch(self.table, self.stride, self.starts, self.lens, self.slots, self.rows, self.room)

    def set_input(self, x) -> None:
        self._set(self.x, np.asarray(x, np.float32).reshape(self.rows, self.width))

    def encode(self) -> None:
        """The blocks over the rows of self.x, to self.y; the slots' sequences are longer by their rows afterwards, unless
        there is no room for them."""
        T, E = self.rows, self.width
        if T == 0:
            return
        ok = g.sessionCacheGrow(gbHip, self.pool, self.all_rows, self.add, self.slots)
        ok &= g.sessionNormBlock(gbHip, self.x, T, E, None, None, None, 1.0, self.h, self.norms[0], self.y)
        for (wq, wk, wv, wo), cache, norm in zip(self.layers, self.caches, self.norms[1:]):
            ok &= g.sessionMatmulQ4(gbHip, self.y, wq, self.q, T)
            ok &= g.sessionMatmulQ4(gbHip, self.y, wk, self.k, T)
            ok &= g.sessionMatmulQ4(gbHip, self.y, wv, self.v, T)
            ok &= g.sessionRopeAppend(gbHip, self.q, self.k, self.v, self.heads, self.rope, cache, self.batch, self.q_rot)
            ok &= g.sessionPagedAttention(gbHip, self.q_rot, self.heads, self.attn, cache, self.batch, self.a)
            ok &= g.sessionMatmulQ4(gbHip, self.a, wo, self.o, T)
            ok &= g.sessionNormBlock(gbHip, self.o, T, E, None, None, self.h, 1.0, self.h, norm, self.y)
        self._taken(ok)

    def _taken(self, ok: bool) -> None:
        if not ok:
            raise _abi.HipUnsupported(f"PagedDecoder: an operator does not take these sizes ({g.sessionGetLastError(gbHip)})")

    def forward(self, x, counts) -> np.ndarray:
        self.set_rows(counts)
        self.set_input(x)
        self.encode()
        return self.output()

    def output(self) -> np.ndarray:
        return g.sessionRead(gbHip, self.y, self.rows * self.width).reshape(self.rows, self.width)

    def record(self) -> int:
        """Keeps a step of the rows last set as a recording; it has been run once."""
        if not g.sessionBeginRecording(gbHip):
            raise _abi.HipBackendError(g.sessionGetLastError(gbHip))
        try:
            self.encode()
        except _abi.HipBackendError:
            g.sessionRecoverQueue(gbHip)
            raise
        if not g.sessionEnd(gbHip):
            raise _abi.HipBackendError(g.sessionGetLastError(gbHip))
        return g.sessionLastRecording(gbHip)

    def fork(self, parents, rows) -> None:
        if len(parents) != len(rows):
            raise ValueError(f"{len(rows)} forks of {len(parents)} parents")
        self._set(self.some, np.asarray(parents, np.int32))
        self._set(self.others, np.asarray(rows, np.int32))
        self._taken(g.sessionCacheFork(gbHip, self.pool, self.some, self.others, len(rows)))

    def free(self, rows) -> None:
        self._set(self.some, np.asarray(rows, np.int32))
        self._taken(g.sessionCacheFree(gbHip, self.pool, self.some, len(rows)))

    def compact(self) -> None:
        self._taken(g.sessionCacheCompact(gbHip, self.pool))

    def lengths(self) -> np.ndarray:
        return g.sessionRead(gbHip, self.lens, self.slots).view(np.int32)

    def granted(self) -> np.ndarray:
        """The tokens that each slot's last step took: its rows, or 0 where there was no room for them."""
        return g.sessionRead(gbHip, self.room, self.slots).view(np.int32)

    def refused(self) -> int:
        """How many times a slot found no room for its rows, since the start."""
        return int(g.sessionRead(gbHip, self.status, 4).view(np.int32)[0])


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__)
    p.add_argument("--layers", type=int, default=4)
    p.add_argument("--width", type=int, default=2048)
    p.add_argument("--heads", type=int, default=16)
    p.add_argument("--kv-heads", type=int, default=4)
    p.add_argument("--head-dim", type=int, default=128)
    p.add_argument("--prompts", type=int, default=4)
    p.add_argument("--beams", type=int, default=4)
    p.add_argument("--prompt-len", type=int, default=900)
    p.add_argument("--steps", type=int, default=64)
    args = p.parse_args()
    rng = np.random.default_rng(0)
    g.ensureGpuInit(gbHip)
    q, kv = args.heads * args.head_dim, args.kv_heads * args.head_dim
    layers = [(random_weights(rng, args.width, q), random_weights(rng, args.width, kv), random_weights(rng, args.width, kv),
               random_weights(rng, q, args.width)) for _ in range(args.layers)]
    norms = [np.ones(args.width, np.float32)] * (args.layers + 1)
    slots = args.prompts * args.beams
    max_len = args.prompt_len + args.steps + 2
    d = PagedDecoder(layers, norms, args.width, args.heads, args.kv_heads, args.head_dim, slots, max_len,
                     args.prompts * args.prompt_len, slots * -(-max_len // 32))
    counts = [0] * slots
    counts[::args.beams] = [args.prompt_len - 37 * i for i in range(args.prompts)]
    t = time.perf_counter()
    d.forward(rng.standard_normal((sum(counts), args.width)), counts)
    print(f"prompts: {sum(counts)} rows in {1e3 * (time.perf_counter() - t):.2f} ms (with their upload and the first launches)", flush=True)
    rows = [i for i in range(slots) if i % args.beams]
    d.fork([i - i % args.beams for i in rows], rows)
    d.set_rows([1] * slots)
    d.set_input(rng.standard_normal((slots, args.width)))
    step = d.record()
    t = time.perf_counter()
    if not g.sessionReplay(gbHip, step, args.steps):
        raise SystemExit(g.sessionGetLastError(gbHip))
    t = (time.perf_counter() - t) / args.steps
    print(f"beams: {slots} rows a step, {1e6 * t:.1f} us a step of {args.layers} layers ({slots / t:.0f} rows/s), lengths {d.lengths().tolist()}", flush=True)
    d.free([i for i in range(slots) if i % args.beams])
    d.compact()
    print(f"one beam each after compaction: lengths {d.lengths().tolist()}, refused {d.refused()}", flush=True)
    g.sessionFreeRecording(gbHip, step)


if __name__ == "__main__":
    main()
