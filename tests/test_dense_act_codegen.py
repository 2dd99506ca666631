"""What the kernels of the dense product with an epilogue rely on, checked in the generated code: the transfers into LDS keep their address in m0, where nothing else may
lie, and nothing that a lane holds is spilled."""

import re
import shutil
import subprocess

import pytest

from neuropress_amd import build


@pytest.mark.parametrize("source, kernel, count, transfers",
                         [("dense_act.hip", "dense_some_kernel", 2 * (2 * 2 + 2), True), ("dense_act.hip", "dense_few_kernel", 2 * 3 * 2, False),
                          ("wide_gemm_epilogue.hip", "wide_gemm_kernel", 2 * 13, True)])  # fmt: skip
def test_m0_is_the_transfers_own_and_nothing_spills(tmp_path, source, kernel, count, transfers):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not build.Path(hipcc).exists():
        pytest.skip("needs hipcc")
    out = tmp_path / "kernels.s"
    res = subprocess.run([hipcc, *build.CXXFLAGS, *build.DEVICE_FLAGS, "-S", "--cuda-device-only", str(build.CSRC / source), "-o", str(out)],
                         capture_output=True, text=True)  # fmt: skip
    assert res.returncode == 0, res.stderr[-2000:]
    text = out.read_text()
    lines = text.split("\n")
    starts = [i for i, ln in enumerate(lines) if re.match(rf"^_ZN\S*{kernel}\S*: *;", ln)]
    assert len(starts) == count
    for i in starts:
        body = lines[i : next(j for j in range(i, len(lines)) if lines[j].startswith(".Lfunc_end"))]
        for k, ln in enumerate(body):  # the three instructions of a transfer, and no other
            if re.search(r"\bm0\b", ln):
                assert re.match(r"\s+s_mov_b32 m0, ", ln) and re.match(r"\s+s_nop 0", body[k + 1]) and "global_load_lds_dword" in body[k + 2], body[k : k + 3]
        assert any("global_load_lds_dwordx4" in ln for ln in body) == transfers == any("v_mfma_f32_16x16x32" in ln for ln in body)
        assert not any(re.match(r"\s+scratch_", ln) for ln in body)
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text)
