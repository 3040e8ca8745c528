"""Plans of many assignments, on both sides of each way of making them (one block, sums formed by every block, sums formed once) and up to the largest the call takes."""
import numpy as np
import pytest

from bybylang_amd import synth
from bybylang_amd import _abi
from test_experts_block_gpu import gb  # noqa: F401
from test_moe_gpu import new_plan, read_plan

pytestmark = pytest.mark.gpu


def check(hip, T, k, E, ids):
    buf, p = new_plan(hip, T, k, E)
    hip.moe_plan(hip.DeviceBuffer.from_array(ids), p)
    agree(buf, T, k, E, ids)


def agree(buf, T, k, E, ids):
    offsets, order = read_plan(buf, T, k, E)
    flat = ids.reshape(-1)
    key = np.where((flat >= 0) & (flat < E), flat, E)
    want = np.argsort(key.astype(np.int16), kind="stable")
    count = np.bincount(key, minlength=E + 1)[:E]
    assert np.array_equal(offsets, np.concatenate([[0], np.cumsum(count)]))
    assert np.array_equal(order[:offsets[-1]], want[:offsets[-1]])


@pytest.mark.parametrize("rows", [4095, 4096, 4097, 65535, 65536, 65537, 67585, 262145, 400001])
@pytest.mark.parametrize("E", [1, 63, 65, 256, 1000, 1024])
def test_sizes(hip, rows, E):
    ids = synth.rng(rows + E).integers(-1, E + 1, (rows, 1)).astype(np.int32)
    check(hip, rows, 1, E, ids)


@pytest.mark.parametrize("T,k,E", [(262144, 8, 256), (70001, 3, 160), (2**24 - 1, 1, 40)])
def test_many(hip, T, k, E):
    g = synth.rng(T)
    check(hip, T, k, E, np.minimum(g.integers(0, E, (T, k)), g.integers(0, E, (T, k))).astype(np.int32))


def test_all_in_one_expert(hip):
    check(hip, 300000, 1, 300, np.full((300000, 1), 299, np.int32))
    check(hip, 300000, 1, 300, np.full((300000, 1), -1, np.int32))


@pytest.mark.parametrize("direct", [0, 1])
@pytest.mark.parametrize("T,E", [(70000, 1024), (9000, 40)])
def test_recorded(hip, gb, direct, T, E):  # noqa: F811
    """A recorded plan follows the ids of each replay, with a plan of another size between."""
    _abi.check(_abi.load().byhip_session_set_direct_replay(direct))
    g = synth.rng(T)
    all_ids = [g.integers(0, E, (T, 1)).astype(np.int32) for _ in range(3)]
    ids = hip.DeviceBuffer.from_array(all_ids[0])
    buf, p = new_plan(hip, T, 1, E)
    assert gb.sessionBeginRecording(gb.gbHip)
    hip.moe_plan(ids, p)
    assert gb.sessionEnd(gb.gbHip)
    step = gb.sessionLastRecording(gb.gbHip)
    for turn in range(2):
        for now in all_ids:
            ids.upload(now)
            check(hip, 5000, 2, 30, g.integers(0, 30, (5000, 2)).astype(np.int32))
            assert gb.sessionReplay(gb.gbHip, step, 1)
            agree(buf, T, 1, E, now)
    gb.sessionFreeRecording(gb.gbHip, step)


def test_units_of_a_large_plan(hip):
    """The products' units cover each expert's rows: outputs of ones count their inputs."""
    T, E, K, N = 200000, 50, 32, 32
    ids = (synth.rng(5).integers(0, E, (T, 1))).astype(np.int32)
    up = hip.DeviceBuffer.from_array
    buf, p = new_plan(hip, T, 1, E)
    hip.moe_plan(up(ids), p)
    x = np.concatenate([np.full(T * K // 2, 0x22, np.uint8), np.full(T, 127, np.uint8)])                        # ones
    w = np.concatenate([np.full(E * N * K // 2, 0x22, np.uint8), np.repeat(127 + np.arange(E) % 9, N).astype(np.uint8)])  # 2^(expert % 9)
    y = up(np.zeros(T * N, np.float32))
    hip.moe_matmul(up(x), _abi.MXFP4_KM, up(w), p, K, N, _abi.MOE_SCATTER, y, N, _abi.F32)
    assert np.array_equal(y.read(np.float32).reshape(T, N), np.repeat(32 * 2.0 ** (ids % 9), N, axis=1))
