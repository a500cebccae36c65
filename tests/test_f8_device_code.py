"""Checks on the device code that hipcc makes of the 8-bit GEMM.

Its e4m3 MFMAs are inline asm, so the compiler does not insert the wait states
that a read of their result needs; whether every read keeps them is a property of
the generated code, looked at here (no GPU needed).
"""

import re
import shlex
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "tiktok-techjam-2026_amd" / "csrc"
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
# wait states between a 16-pass MFMA (32x32x64, e4m3) and another instruction's
# use of its result on gfx950
RESULT_STATES = 20


def _vgprs(text):
    regs = set()
    for lo, hi, one in re.findall(r"\bv(?:\[(\d+):(\d+)\]|(\d+)\b)", text):
        regs |= set(range(int(lo), int(hi) + 1)) if lo else {int(one)}
    return regs


def _operands(line):
    return [t.strip() for t in re.split(r",(?![^\[]*\])", line.split(None, 1)[1])] if " " in line else []


def _early_uses(code):
    """(MFMA, instruction) pairs where the instruction touches the MFMA's
    result too early, along every path.  An instruction counts as one state,
    s_nop N as N + 1, time spent at a barrier or a wait as none; an MFMA that adds
    to just this result may follow at once, and answers for it from there on."""
    label = {l[:-1]: i for i, l in enumerate(code) if l.endswith(":")}
    bad = []
    for start, mfma in enumerate(code):
        if not mfma.startswith("v_mfma"):
            continue
        dest = _operands(mfma)[0]
        regs = _vgprs(dest)
        paths, seen = [(start + 1, RESULT_STATES)], set()
        while paths:
            i, left = paths.pop()
            while left > 0 and i < len(code) and (i, left) not in seen:
                seen.add((i, left))
                l = code[i]
                if l.endswith(":"):
                    i += 1
                    continue
                ops = _operands(l)
                if l.startswith("v_mfma") and ops[0] == dest and (ops[3] == dest or not _vgprs(ops[3])) \
                        and not (_vgprs(ops[1]) | _vgprs(ops[2])) & regs:
                    break
                if _vgprs(l) & regs:
                    bad.append((mfma, l))
                    break
                left -= int(l.split()[1]) + 1 if l.startswith("s_nop") else 0 if l.startswith(("s_wait", "s_barrier")) else 1
                if l.startswith("s_endpgm"):
                    break
                if l.startswith(("s_branch", "s_cbranch")):
                    paths.append((label[l.split()[1]], left))
                    if l.startswith("s_branch"):
                        break
                i += 1
    return bad


def test_early_use_is_found():
    k0, k1 = "v_mfma_f32_32x32x64_f8f6f4 v[0:15], v[16:23], v[24:31], 0", \
             "v_mfma_f32_32x32x64_f8f6f4 v[0:15], v[16:23], v[24:31], v[0:15]"
    read = "v_fma_f32 v40, v3, v41, v40"
    assert not _early_uses([k0, k1, "s_nop 15", "s_nop 3", read])
    assert _early_uses([k0, k1, "s_nop 15", "s_nop 2", read])
    assert _early_uses([k0, k1, "s_nop 15", "s_waitcnt vmcnt(0)", "s_barrier", read])
    assert _early_uses([k0, "v_mov_b32_e32 v50, v15"])
    assert _early_uses(["L:", read, "s_nop 15", k1, "s_cbranch_scc1 L"])
    assert not _early_uses([k1, "v_fma_f32 v40, v16, v41, v40"])


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if not Path(HIPCC).exists() or shutil.which("make") is None:
        pytest.skip("needs hipcc and make")
    made = subprocess.run(["make", "-n", "-B", "-C", str(CSRC), "../../_build/tjk/gemm_f8.o"], check=True,
                          capture_output=True, text=True).stdout
    line = next(l for l in made.splitlines() if " -c " in l)
    out = tmp_path_factory.mktemp("f8") / "gemm_f8.s"
    subprocess.run([HIPCC, *shlex.split(line.split(" -c ")[0])[1:], "--cuda-device-only", "-S", str(CSRC / "gemm_f8.hip"),
                    "-o", str(out)], check=True, capture_output=True)
    asm, found = out.read_text(), {}
    for m in re.finditer(r"^(_ZN3tjk14gemm_f8_kernel\S+):", asm, re.M):
        body = asm[m.end():asm.index(".Lfunc_end", m.end())]
        lines = [l.split(";")[0].strip() for l in body.splitlines()]
        found[m.group(1)] = [l for l in lines if l and (not l.startswith(".") or l.endswith(":"))]
    return found


def test_gemm_f8_reads_products_after_their_wait(kernels):
    """Every instance: no read or copy of a product before its MFMAs are done,
    and no scratch (a spilled product is such a read)."""
    assert len(kernels) == 9 * 4 + 3 * 2  # tiles x (two 2-byte types x GELU or not), x (e4m3 x GELU or not)
    for name, code in kernels.items():
        assert sum(l.startswith("v_mfma") for l in code) >= 4, name
        e4m3 = {"f8f6f4" in l for l in code if l.startswith("v_mfma")}
        assert len(e4m3) == 1, name
        if True in e4m3:  # the others' waits are the compiler's
            assert not _early_uses(code), (name, _early_uses(code)[:3])
        assert not any(l.startswith("scratch_") for l in code), name


def test_gemm_f8_operands_are_not_just_written(kernels):
    """No vector instruction writes an MFMA's operand in the four before it:
    operands come from LDS, behind a wait."""
    for name, code in kernels.items():
        code = [l for l in code if not l.startswith("s_wait")]
        for i, l in enumerate(code):
            if l.startswith("v_mfma") and "f8f6f4" in l:
                regs = _vgprs(_operands(l)[1]) | _vgprs(_operands(l)[2])
                for b in code[max(0, i - 4):i]:
                    if b.startswith("v_") and not b.startswith("v_mfma"):
                        assert not _vgprs(_operands(b)[0]) & regs, (name, b, l)


def test_gemm_f8_stays_off_packed_fp32(kernels):
    for name, code in kernels.items():
        assert not any(re.match(r"v_pk_(add|mul|fma)_f32", l) for l in code), name
