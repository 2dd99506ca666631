"""What the layer norm's kernels and the epilogue forms of the dense product's narrow tiles hold stays in registers, checked in the generated code."""

import re
import shutil
import subprocess

import pytest

from neuropress_amd import build


# layer norm, a type each: eleven forms of rows in registers, rows of a block's own; backward: one and two pieces to a lane, a block's own, columns, the parts' sums
@pytest.mark.parametrize("source, kernel, count", [("layer_norm.hip", r"layer_norm_\w*_kernel", 3 * (11 + 1 + 2 + 1 + 1 + 1)),
                                                   ("dense_gemm.hip", r"dense_gemm_kernelILi[01](?:ELi\d)+ELb[01]ELb1E|splitk_reduce_epilogue_kernel", 2 * (2 * 2 + 1))])  # fmt: skip
def test_nothing_spills(tmp_path, source, kernel, count):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not build.Path(hipcc).exists():
        pytest.skip("needs hipcc")
    out = tmp_path / "kernels.s"
    res = subprocess.run([hipcc, *build.CXXFLAGS, *build.DEVICE_FLAGS, "-S", "--cuda-device-only", str(build.CSRC / source), "-o", str(out)],
                         capture_output=True, text=True)  # fmt: skip
    assert res.returncode == 0, res.stderr[-2000:]
    text = out.read_text()
    lines = text.split("\n")
    starts = [i for i, ln in enumerate(lines) if re.match(rf"^_ZN\S*(?:{kernel})\S*: *;", ln)]
    assert len(starts) == count
    for i in starts:
        body = lines[i : next(j for j in range(i, len(lines)) if lines[j].startswith(".Lfunc_end"))]
        assert not any(re.match(r"\s+scratch_", ln) for ln in body), lines[i]
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text)
