"""Attention's workspace: a program without attention does not hold it, and the call that takes it may be the first of a recording."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# A process of its own, because the workspace is taken once. Its argument: whether the first call is recorded for direct replay.
PROGRAM = r"""
import sys
import numpy as np
from bybylang_amd import _abi, device as dev, gpubackend as g
lib = _abi.load()
dev.init(0)
assert lib.byhip_debug_alloc_count() == 2, lib.byhip_debug_alloc_count()  # the GEMMs' workspace and the flags
rng, up = np.random.default_rng(1), dev.DeviceBuffer.from_array
k, v = (up(rng.standard_normal((9, 2, 16, 64)).astype(np.float16)) for _ in range(2))
q = up(rng.standard_normal((3, 4 * 64)).astype(np.float32))
table, lens = up(np.arange(9, dtype=np.int32)), up(np.array([140], np.int32))
starts, out = up(np.array([0, 3], np.int32)), up(np.zeros((3, 4 * 64), np.float32))
cache, batch, attn = dev.KvCache(k, v, dev.F16, 9, 16, 2, 64), dev.KvBatch(table, 9, starts, lens, 1, 3), dev.Attn(0.125)
run = lambda: dev.paged_attention(q, 256, dev.F32, 4, attn, cache, batch, out, 256, dev.F32)
before = lib.byhip_debug_alloc_count()
_abi.check(lib.byhip_session_set_direct_replay(int(sys.argv[1])))
assert g.sessionBeginRecording(g.gbHip)
run()
assert g.sessionEnd(g.gbHip), g.sessionGetLastError(g.gbHip)
kept = g.sessionLastRecording(g.gbHip)
assert lib.byhip_debug_alloc_count() == before + 1
got = []
for i in range(4):  # eager work and other queries between the replays
    q.upload(rng.standard_normal((3, 4 * 64)).astype(np.float32))
    run()
    want = out.read(np.float32)
    out.upload(np.zeros((3, 4 * 64), np.float32))
    assert g.sessionReplay(g.gbHip, kept, 1)
    assert np.array_equal(out.read(np.float32), want) and np.all(want != 0), i
assert lib.byhip_debug_alloc_count() == before + 1
print("fine")
"""


@pytest.mark.parametrize("direct", [0, 1], ids=["graph", "direct"])
def test_the_first_attention_takes_it_also_when_recorded(direct):
    r = subprocess.run([sys.executable, "-c", PROGRAM, str(direct)], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout == "fine\n", r.stdout + r.stderr[-3000:]
