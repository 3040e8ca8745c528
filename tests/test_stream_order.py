"""The library's stream does not wait for the null stream (hipStreamNonBlocking), so nothing in the library may be written on the
null stream: such a write and a kernel that reads it would have no order. CPU only: it reads the sources."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bybylang_amd", "csrc")


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.hip"))), ids=os.path.basename)
def test_nothing_is_written_on_the_null_stream(path):
    text = re.sub(r"//[^\n]*", "", open(path).read())
    assert not re.findall(r"\b(hipMemset(?:D\d+)?|hipMemcpyToSymbol)\s*\(", text)
    assert not re.findall(r"\bhipMemcpy\s*\([^;]*hipMemcpyHostToDevice", text)
    assert "<<<" not in text  # kernels go through launch(), on the library's stream
