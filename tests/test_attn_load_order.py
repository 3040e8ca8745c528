"""attn_chunk counts its direct loads: its barriers wait until all but the newest WAIT of a wave's loads have landed, whose number
the source derives from whole batches. The loads are assembly that the compiler does not count, so what it makes of the loops has
to keep them in whole batches between the barriers that the count was made for, each with its own LDS address in m0. This reads
every compiled instantiation (the objects that the library was linked from), and checks that a listing with a load, a wait or
an address left out would be found. CPU only: it needs the build's objects and binutils."""
import os
import re
import shutil

import pytest

from test_load_order import BUILD, LLVM, listing

ADDRESS = re.compile(r"\bm0, ")


def tokens(lines):
    """X, W: a direct load of 16 or 4 bytes per lane; 'm0': the address register written; an int: a barrier and the vmcnt of the wait right
    before it, None without one."""
    out, wait = [], None
    for line in lines:
        if "global_load_lds_dword" in line:
            out.append("X" if "dwordx4" in line else "W")
        elif ADDRESS.search(line):
            out.append("m0")
        if "s_barrier" in line:
            out.append(("barrier", wait))
        m = re.search(r"s_waitcnt vmcnt\((\d+)\) lgkmcnt\(0\)", line)
        wait = int(m.group(1)) if m else None
    return out


def faults(toks, dim, waves):
    """What in a kernel's tokens its counts do not allow."""
    loads = 128 * dim // 1024 // waves  # of K or V, per wave and tile
    ahead, early = (2 if waves == 8 else 1), dim <= 64
    batch = "X" * 2 * loads + "W"
    prologue, wait = "W" + "X" * loads + batch * ahead, (ahead if early else ahead - 1) * len(batch)
    bad, seen, segment, fresh, began = [], 0, "", False, None
    for t in toks:
        if t == "m0":
            fresh = True
        elif isinstance(t, str):
            if not fresh:
                bad.append("a load without an address of its own")
            fresh, segment = False, segment + t
        else:
            ended = t[1]
            if segment == prologue:
                if began != 0 or ended != ahead * len(batch):
                    bad.append(f"prologue between waits {began} and {ended}")
                seen += 100
            elif segment == batch:
                if (ended if early else began) != wait:
                    bad.append(f"batch between waits {began} and {ended}")
                seen += 1
            elif segment:
                bad.append(f"loads {segment}")
            elif wait and ((ended if early else began) == wait):
                bad.append(f"a wait for all but {wait} loads without a batch beside it")
            segment, began = "", ended
    if segment:
        bad.append("loads after the last barrier")
    if seen < 100 or seen >= 200 or seen % 100 < 4:  # waves without rows, the first tile, the loop, the careful pass
        bad.append(f"{seen // 100} prologues, {seen % 100} batches")
    return bad


@pytest.fixture(scope="module", params=["f16", "bf16"])
def kernels(request, tmp_path_factory):
    path = os.path.join(BUILD, f"byhip_attn_chunk_{request.param}.hip.o")
    if not (os.path.exists(path) and shutil.which("objcopy") and os.path.exists(LLVM + "/llvm-objdump")):
        pytest.skip("the build's objects or binutils are not there")
    out, name = {}, None
    for line in listing(path, tmp_path_factory.mktemp("listing")):
        m = re.match(r"[0-9a-f]+ <(.*)>:", line)
        if m:
            m = re.search(r"10attn_chunkI(.*)EEv", m.group(1))
            name = tuple(int(v) for v in re.findall(r"L[ib](\d+)E", m.group(1) + "E")) if m else None
            if name:
                out[name] = []
        elif name:
            out[name].append(line)
    return {n: tokens(lines) for n, lines in out.items()}


def test_loads_stand_in_whole_batches_between_their_barriers(kernels):
    assert len(kernels) == 16
    for (_, _, dim, _, waves, _), toks in kernels.items():
        assert faults(toks, dim, waves) == [], (dim, waves)


def test_what_is_left_out_is_found(kernels):
    for (_, _, dim, _, waves, _), toks in kernels.items():
        first = next(i for i, t in enumerate(toks) if t in ("X", "W"))
        for i in range(first - 1, len(toks)):
            if isinstance(toks[i], tuple):
                if not toks[i][1]:
                    continue
                planted = toks[:i] + [("barrier", toks[i][1] + 1)] + toks[i + 1:]
            else:
                if toks[i] == "m0" and toks[i - 1] == "m0" or toks[i] == "m0" and toks[i + 1] == "m0":
                    continue
                planted = toks[:i] + toks[i + 1:]
            assert faults(planted, dim, waves), (dim, waves, i, toks[i])
