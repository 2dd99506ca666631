"""What the kernels of the mixture-of-experts layer rely on, checked in the generated code: the transfers into LDS keep their address in m0, where nothing else may lie,
and a step's operands stay in registers."""

import re
import shutil
import subprocess

import pytest

from neuropress_amd import build


def test_m0_is_the_transfers_own_and_nothing_spills(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not build.Path(hipcc).exists():
        pytest.skip("needs hipcc")
    out = tmp_path / "moe.s"
    res = subprocess.run([hipcc, *build.CXXFLAGS, *build.DEVICE_FLAGS, "-S", "--cuda-device-only", str(build.CSRC / "moe.hip"), "-o", str(out)],
                         capture_output=True, text=True)  # fmt: skip
    assert res.returncode == 0, res.stderr[-2000:]
    text = out.read_text()
    lines = text.split("\n")
    starts = [i for i, ln in enumerate(lines) if re.match(r"^_ZN\S*moe_(up|down)_kernel\S*: *;", ln)]
    assert len(starts) == 2 * 3 * (1 + 2 * 2 * 3)  # activation types; up (two forms) and down; dense, 4 and 8 bits with and without zero points and three kinds of groups
    for i in starts:
        body = lines[i : next(j for j in range(i, len(lines)) if lines[j].startswith(".Lfunc_end"))]
        for k, ln in enumerate(body):  # the three instructions of a transfer, and no other
            if re.search(r"\bm0\b", ln):
                assert re.match(r"\s+s_mov_b32 m0, ", ln) and re.match(r"\s+s_nop 0", body[k + 1]) and "global_load_lds_dword" in body[k + 2], body[k : k + 3]
        assert any("global_load_lds_dwordx4" in ln for ln in body) and any("v_mfma_f32_16x16x32" in ln for ln in body)
        assert not any(re.match(r"\s+scratch_", ln) for ln in body)
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text)
