"""What the block-scaled product's kernels keep in LDS lies inside what they
declare (no GPU: the layout is worked out from the tile's parameters, the size
is read from the code that hipcc makes)."""

import re
import shlex
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "tiktok-techjam-2026_amd" / "csrc"
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


@pytest.fixture(scope="module")
def declared(tmp_path_factory):
    """LDS bytes that each instance declares, by its mangled name."""
    if not Path(HIPCC).exists() or shutil.which("make") is None:
        pytest.skip("needs hipcc and make")
    made = subprocess.run(["make", "-n", "-B", "-C", str(CSRC), "../../_build/tjk/gemm_f8.o"], check=True,
                          capture_output=True, text=True).stdout
    line = next(l for l in made.splitlines() if " -c " in l)
    out = tmp_path_factory.mktemp("f8") / "gemm_f8.s"
    subprocess.run([HIPCC, *shlex.split(line.split(" -c ")[0])[1:], "--cuda-device-only", "-S", str(CSRC / "gemm_f8.hip"),
                    "-o", str(out)], check=True, capture_output=True)
    return {name: int(size) for name, size in
            re.findall(r"\.amdhsa_kernel (_ZN3tjk14gemm_f8_kernel\S+)\s+\.amdhsa_group_segment_fixed_size (\d+)",
                       out.read_text())}


def _written(fm, fn, wm, wn, groups, ra, rw, bias_bytes):
    """The end of what a kernel writes: per K group the panels' rings (32 rows
    of 128 bytes a wave row or column), the scales of 8 K tiles of every row and of
    the weights (two loads of 64 words); over them the groups' sums, in rows
    with four floats between them; behind both the tile's bias, which whole loads
    of 64 words bring."""
    bm, bn = 32 * fm * wm, 32 * fn * wn
    group = 4096 * (ra * wm + rw * wn) + 8 * bm * 4 + 512
    sums = groups * bm * (bn + 4) * 4 if groups > 1 else 0
    return max(groups * group, sums) + -(-bn * bias_bytes // 256) * 256


def test_lds_holds_what_is_written(declared):
    assert len(declared) == 9 * 4 + 3 * 2
    for name, size in declared.items():
        # <type of the bias, GELU, e4m3 output, F8Geom<FM, FN, WM, WN, KG, RA, RW, ...>>
        geom = [int(v) for v in re.findall(r"Li(\d+)E", name.split("F8GeomI")[1])[:7]]
        bias_bytes = 4 if re.match(r"_ZN3tjk14gemm_f8_kernelIf", name) else 2
        assert _written(*geom, bias_bytes) <= size <= 160 * 1024, (name, geom, size)
