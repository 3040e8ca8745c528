"""PagedDecoder refuses blocks of experts that do not fit it before anything is made (no GPU)."""
import pytest

from bybylang_amd import gpubackend as g
from bybylang_amd.paged_decoder import PagedDecoder


class Block:
    def __init__(self, width, max_rows):
        self.width, self.max_rows = width, max_rows


@pytest.mark.parametrize("experts,match", [([Block(64, 16)], "1 blocks of experts for 2 layers"), ([Block(64, 16)] * 3, "3 blocks of experts"), ([None, Block(96, 16)], "of 96 values"),
                                           ([Block(64, 15), None], "over 15 rows")])
def test_blocks_that_do_not_fit(monkeypatch, experts, match):
    """A list of another length left layers out of every step."""
    for proc in ("sessionAllocScratch", "sessionUpload"):
        monkeypatch.setattr(g, proc, lambda *a: pytest.fail("allocated"))
    with pytest.raises(ValueError, match=match):
        PagedDecoder([(None,) * 4] * 2, [None] * 3, 64, 4, 2, 16, 2, 32, 16, 8, 16, experts=experts)
