"""Counts near 2^31 in the calls over a paged cache are refused, not wrapped round."""
import numpy as np
import pytest

from bybylang_amd import _abi

pytestmark = pytest.mark.gpu
F16 = _abi.F16


class Elsewhere:
    """Memory that is not the library's, whose size it does not know."""
    ptr = 1 << 20


def pool(hip, lens, cols, page, pages=1):
    up = hip.DeviceBuffer.from_array
    kv = [up(np.zeros(pages * page, np.float16)) for _ in range(2)]
    b = {"table": up(np.full((len(lens), cols), -1, np.int32)), "lens": up(np.array(lens, np.int32)), "refs": up(np.zeros(pages, np.int32)),
         "status": up(np.zeros(4, np.int32))}
    return b, hip.KvPool([hip.KvCache(*kv, F16, pages, page, 1, 1)], b["refs"], b["table"], cols, b["lens"], len(lens), b["status"])


def test_lengths_past_31_bits_are_refused(hip):
    up = hip.DeviceBuffer.from_array
    most = 2**31 - 1
    b, p = pool(hip, [most - 1, most, 5, 0], 4096, 2**20)  # the table has room for 2^32 tokens
    hip.cache_grow(p, up(np.array([0, 1, 2, 3], np.int32)), up(np.array([5, 1, most, 7], np.int32)), 4)
    assert b["lens"].read(np.int32).tolist() == [most - 1, most, 5, 7]
    assert b["status"].read(np.int32).tolist() == [3, 0, 0, 1]
    assert b["refs"].read(np.int32).tolist() == [1]
    table = b["table"].read(np.int32).reshape(4, -1)
    assert table[3, 0] == 0 and (table >= 0).sum() == 1


def test_more_pages_than_are_counted_are_refused(hip):
    b, p = pool(hip, [0], 4, 16)
    far = Elsewhere()
    wide = hip.KvPool(p.keep[1], b["refs"], far, 2**21, far, 1024, b["status"])  # 1024 slots that may ask for 2^31 pages
    with pytest.raises(_abi.HipUnsupported, match="1024 slots of 2097152 pages"):
        hip.cache_grow(wide, far, far, 1024)


def test_more_rows_than_are_counted_are_refused(hip):
    far, ints = Elsewhere(), hip.DeviceBuffer.from_array(np.zeros(8, np.int32))
    with pytest.raises(_abi.HipUnsupported, match="268435457 rows of 16 heads over 2"):
        hip.paged_attention(far, 128, F16, 16, hip.Attn(0.1), hip.KvCache(far, far, F16, 2, 4, 2, 8), hip.KvBatch(ints, 4, ints, ints, 1, 2**28 + 1), far, 128, F16)
