"""Checks on the device code that hipcc makes of the tree attention.

Its copies into LDS are inline asm, into which the compiler does not look for wait
states: whether a vector memory instruction finds its SGPRs settled is a property
of the generated code, looked at here (no GPU needed).  A descriptor whose size
was written by v_readfirstlane one instruction ahead has faulted the GPU.
"""

import re
import shutil
from pathlib import Path

import pytest

from test_device_code import LIB, OBJDUMP, _library_kernels

SGPR_STATES = 5  # between a VALU write of an SGPR and vector memory that reads it


def _sgprs(text):
    regs = set()
    for lo, hi, one in re.findall(r"\bs(?:\[(\d+):(\d+)\]|(\d+)\b)", text):
        regs |= set(range(int(lo), int(hi) + 1)) if lo else {int(one)}
    return regs


def _early_reads(code):
    """(write, read) pairs of a VALU write of an SGPR and a vector memory
    instruction that reads it too soon, and of a write of m0 next to a copy into
    LDS.  (Along the code as it lies: a copy's asm holds its waits itself.)"""
    bad = []
    for i, l in enumerate(code):
        if not l.startswith(("buffer_", "global_", "scratch_")):
            continue
        if l.endswith("lds") and i and re.match(r"s_\w+ m0\b", code[i - 1]):
            bad.append((code[i - 1], l))
        left, j = SGPR_STATES, i - 1
        while left > 0 and j >= 0:
            p = code[j]
            if p.startswith("v_") and " " in p and _sgprs(p.split(None, 1)[1].split(",")[0]) & _sgprs(l):
                bad.append((p, l))
                break
            left -= int(p.split()[1]) + 1 if p.startswith("s_nop") else 1
            j -= 1
    return bad


def test_early_read_is_found():
    copy = "buffer_load_dwordx4 v1, s[4:7], 0 offen lds"
    assert _early_reads(["v_readfirstlane_b32 s6, v2", copy])
    assert _early_reads(["v_readlane_b32 s4, v2, 3", "s_nop 3", copy])
    assert _early_reads(["s_mov_b32 m0, s9", copy])
    assert not _early_reads(["v_readlane_b32 s4, v2, 3", "s_nop 4", "s_mov_b32 m0, s9", "s_nop 0", copy])
    assert not _early_reads(["v_readlane_b32 s8, v2, 3", copy]) and not _early_reads(["s_mov_b32 s4, s9", copy])


@pytest.mark.skipif(not Path(OBJDUMP).exists() or not LIB.exists() or shutil.which("make") is None,
                    reason="needs llvm-objdump and the built library")
def test_copies_find_their_descriptors_settled(tmp_path):
    kernels = dict(_library_kernels(tmp_path, LIB, "tree_attention_kernel"))
    assert len(kernels) >= 8
    for name, code in kernels.items():
        assert sum(l.endswith("lds") for l in code) >= 6, name
        assert not _early_reads(code), (name, _early_reads(code)[:3])
