"""Inline assembly in the kernels names no register that the compiler has not been told of: what a statement reads or writes is an
operand of it ("v", "s", "{m0}") or on its clobber list. m0 and vcc, which the compiler uses for purposes of its own, cannot be
named as clobbered, so they may only be operands. CPU only: it reads the sources."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bybylang_amd", "csrc")


def statements(text):
    """(template string, the rest) of every asm statement."""
    for m in re.finditer(r"\basm\b\s*(?:volatile)?\s*\(((?:\s*\"(?:[^\"\\]|\\.)*\")+)(.*?)\)\s*;", text, re.S):
        yield "".join(re.findall(r"\"((?:[^\"\\]|\\.)*)\"", m.group(1))), m.group(2)


def named(template):
    return set(re.findall(r"(?<![\w%])(m0|vcc(?:_lo|_hi)?|exec(?:_lo|_hi)?|scc|[vsa]\d+|[vsa]\[\d+:\d+\])(?!\w)", template))


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.hip"))), ids=os.path.basename)
def test_registers_are_operands(path):
    for template, _ in statements(open(path).read()):
        assert not named(template), template


def test_named_registers_are_seen():
    found = list(statements('asm volatile("s_mov_b32 m0, %1\\n\\tglobal_load_lds_dword %0, off" ::"v"(p), "s"(to) : "memory");'))
    assert [named(t) for t, _ in found] == [{"m0"}]
    assert not named('s_waitcnt vmcnt(%0) lgkmcnt(0)\\n\\ts_barrier') and named("v_add_f32 v3, %0, v[4:5]") == {"v3", "v[4:5]"}
