"""byhip_paged_attention at the ends of its numbers: empty and tiny queries."""
import numpy as np
import pytest

from bybylang_amd import _abi
from test_attn_gpu import Case

pytestmark = pytest.mark.gpu
F32, F16, BF16 = _abi.F32, _abi.F16, _abi.BF16


@pytest.mark.parametrize("new", [1, 20, 200])
@pytest.mark.parametrize("ct", [F16, BF16])
@pytest.mark.parametrize("scale", [None, 2.0**-11, 1e-20, 1e-38])
@pytest.mark.parametrize("value", [0.0, 1e-42, 1e-38, 1e-30])
def test_empty_and_tiny_queries(hip, new, ct, scale, value):
    """Rows of padding have queries of zeros: they weigh the keys that they see alike, and no others."""
    c = Case(hip, [230], [new], 4, 2, 128, 32, ct, F32, F32, seed=20, scale=scale)
    c.q[::2] = np.float32(value) * np.sign(c.q[::2])
    c.check()
