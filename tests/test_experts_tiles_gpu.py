"""The block of experts recorded at sizes whose products run in moe_tiles, and whose plan is of many blocks: replays against eager calls bit for bit."""
import numpy as np
import pytest

from bybylang_amd import _abi
from test_experts_block_gpu import Block, gb  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("direct", [0, 1])
def test_recorded(gb, direct):  # noqa: F811
    _abi.check(_abi.load().byhip_session_set_direct_replay(direct))
    D, F, E, k, T = 1024, 1408, 4, 2, 2500
    b = Block(gb, D, F, E, k, T)
    handles = [gb.sessionUpload(gb.gbHip, np.zeros(T * D, np.float32)) for _ in range(2)]
    out = gb.sessionAllocScratch(gb.gbHip, T * D)

    def put(arrays):
        for handle, a in zip(handles, arrays):
            a = np.ascontiguousarray(a, np.float32)
            _abi.check(_abi.load().byhip_upload(handle.ptr, 0, a.ctypes.data, a.nbytes))
    inputs = [(b.rng.standard_normal((T, D)), b.rng.standard_normal((T, D)) * 10.0**i) for i in range(3)]
    want = []
    for pair in inputs:
        put(pair)
        assert b.block.encode(handles[0], T, handles[1], out)
        want.append((b.floats(out, T, D), b.floats(handles[1], T, D), b.floats(b.block.ids, T, k)))
        assert np.isfinite(want[-1][0]).all() and want[-1][0].any()
    assert not np.array_equal(want[0][2], want[1][2])
    other = [gb.sessionUpload(gb.gbHip, b.rng.standard_normal(700 * D).astype(np.float32)) for _ in range(3)]
    assert gb.sessionBeginRecording(gb.gbHip)
    assert b.block.encode(handles[0], T, handles[1], out)
    assert gb.sessionEnd(gb.gbHip)
    step = gb.sessionLastRecording(gb.gbHip)
    for turn in range(2):
        for pair, (o, h, ids) in zip(inputs, want):
            put(pair)
            assert b.block.encode(other[0], 700, other[1], other[2])
            assert gb.sessionReplay(gb.gbHip, step, 1)
            assert np.array_equal(b.floats(out, T, D).view(np.uint32), o.view(np.uint32))
            assert np.array_equal(b.floats(handles[1], T, D), h) and np.array_equal(b.floats(b.block.ids, T, k).view(np.int32), ids.view(np.int32))
    gb.sessionFreeRecording(gb.gbHip, step)
