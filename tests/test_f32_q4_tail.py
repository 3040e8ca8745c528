"""gemm_f32_q4 and gemm_planes keep the loads of a step or two in flight by counting them. In their last steps nothing follows that would use loads two steps
ahead; the compiler drops such loads into registers but not those into LDS, so a count of them all lets a barrier pass before the last
step's activations are in LDS. This reads the compiled kernels: the loop's three barriers leave a step's loads in flight, the two of the last steps none; gemm_planes' eight
last steps leave no more than the direct loads of two.
CPU only: it needs the build's objects and binutils."""
import os
import re
import shutil

import pytest

from test_load_order import BUILD, LLVM, listing


def barriers(obj, tmp):
    """{mangled name: the vmcnt that is waited for ahead of each barrier, in the listing's order}"""
    out, name, wait = {}, None, None
    for line in listing(obj, tmp):
        m = re.match(r"[0-9a-f]+ <(.*)>:", line)
        if m:
            name, wait = m.group(1), None
        elif name and line.startswith("\t"):
            m = re.search(r"s_waitcnt.*vmcnt\((\d+)\)", line)
            if m:
                wait = int(m.group(1))
            if "s_barrier" in line:
                out.setdefault(name, []).append(wait)
    return out


def test_last_steps_wait_for_their_activations(tmp_path):
    path = os.path.join(BUILD, "byhip_exact.hip.o")
    if not (os.path.exists(path) and shutil.which("objcopy") and os.path.exists(LLVM + "/llvm-objdump")):
        pytest.skip("the build's objects or binutils are not there")
    seen = 0
    for name, waits in barriers(path, tmp_path).items():
        m = re.search(r"11gemm_f32_q4ILi(\d)ELb(\d)EEEv", name)
        if not m:
            continue
        seen += 1
        loads = int(m.group(1)) + 2 + (1 - int(m.group(2)))
        assert sorted(waits) == [0, 0] + [loads] * 3, f"{name}: {waits}"
    assert seen == 8


def test_guarded_steps_count_direct_loads_only(tmp_path):
    path = os.path.join(BUILD, "byhip_planes.hip.o")
    if not (os.path.exists(path) and shutil.which("objcopy") and os.path.exists(LLVM + "/llvm-objdump")):
        pytest.skip("the build's objects or binutils are not there")
    seen = 0
    for name, waits in barriers(path, tmp_path).items():
        m = re.search(r"11gemm_planesILNS_\w*?BFormatE\dELi(\d)E", name)
        if not m:
            continue
        seen += 1
        few = [w for w in waits if w is not None and w <= 2 * int(m.group(1))]
        assert len(few) >= 8, f"{name}: {waits}"
    assert seen >= 8
