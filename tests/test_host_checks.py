"""Host checks of arguments, built without optimisation: an unknown dtype is answered, not divided by. CPU only: it needs hipcc."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC") or ("/opt/rocm/bin/hipcc" if os.path.exists("/opt/rocm/bin/hipcc") else shutil.which("hipcc"))

PROGRAM = r"""
#include <cstdio>
#include "byhip_cache.h"
int main() {
    float x[8];
    for (int dtype = -1; dtype < 9; ++dtype) std::printf("%d", (int)byhip::aligned4(x + 4 - ((uintptr_t)x / 4) % 4, 64, dtype));
}
"""


def test_alignment_of_unknown_dtypes(tmp_path):
    if not HIPCC:
        pytest.skip("hipcc not available")
    src, exe = tmp_path / "a.hip", tmp_path / "a"
    src.write_text(PROGRAM)
    cmd = [HIPCC, "--offload-arch=gfx950", "--cuda-host-only", "-O0", "-std=c++17", "-I" + os.path.join(ROOT, "include"),
           "-I" + os.path.join(ROOT, "bybylang_amd", "csrc"), str(src), "-o", str(exe)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert (r.returncode, r.stdout) == (0, "0111000000")  # F32, F16, BF16
