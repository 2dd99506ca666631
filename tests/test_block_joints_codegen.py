"""What the kernels that join a block's halves rely on, checked in the generated code: the compiler keeps nothing of its own in m0, which the transfers into LDS write, no vector load of its own is under way
where theirs are counted by hand, and nothing is kept in memory but where a comment says so."""

import re
import shutil
import subprocess

import pytest

from neuropress_amd import build


def _kernels(tmp_path, source, name):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not build.Path(hipcc).exists():
        pytest.skip("needs hipcc")
    out = tmp_path / "kernels.s"
    res = subprocess.run([hipcc, *build.CXXFLAGS, *build.DEVICE_FLAGS, "-S", "--cuda-device-only", str(build.CSRC / source), "-o", str(out)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
    text = out.read_text()
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text)
    lines = text.split("\n")
    for i in (i for i, ln in enumerate(lines) if re.match(rf"^_ZN\S*(?:{name})\S*: *;", ln)):
        body = lines[i : next(j for j in range(i, len(lines)) if lines[j].startswith(".Lfunc_end"))]
        yield lines[i].split(":")[0], [ln.split(";")[0] for ln in body]


def _m0_is_the_transfers(code):
    return not [ln for ln in code if re.search(r"\bm0\b", ln) and not re.match(r"\s+s_mov_b32 m0, s\d+", ln)]


def _spills(code):
    return [ln for ln in code if re.match(r"\s+scratch_", ln)]


@pytest.mark.parametrize("source,count", [("wide_gemm_gated.hip", 2 * 9), ("wide_gemm_turned.hip", 2 * 2 * 5)])
def test_wide_tiles(tmp_path, source, count):
    kernels = list(_kernels(tmp_path, source, "wide_gemm_kernel"))
    assert len(kernels) == count
    for name, code in kernels:
        assert _m0_is_the_transfers(code) and not _spills(code), name
        first = next(k for k, ln in enumerate(code) if "global_load_lds" in ln)
        last = max(k for k, ln in enumerate(code) if "v_mfma" in ln)
        loop = code[first : last + 1]
        assert not [ln for ln in loop if re.search(r"v_accvgpr_(mov|read|write)", ln)], name
        assert not [ln for ln in loop if re.search(r"global_load_(?!lds)|flat_load|buffer_load", ln)], name
        if source == "wide_gemm_turned.hip":
            assert [ln for ln in loop if "ds_read_b64_tr_b16" in ln], name


def test_wide_pair(tmp_path):
    kernels = list(_kernels(tmp_path, "wide_gemm_pair.hip", "wide_gemm_pair_kernel"))
    assert len(kernels) == 2 * 5
    for name, code in kernels:
        assert _m0_is_the_transfers(code) and not _spills(code), name
        assert not [ln for ln in code if re.search(r"v_accvgpr_(mov|read|write)", ln)], name


def test_adapters(tmp_path):
    kernels = list(_kernels(tmp_path, "adapters.hip", "adapter_\\w+_kernel"))
    assert len(kernels) == 1 + 2 * (1 + 2 * 3) + 2 * (6 + 5)  # the list; down; up by the ballot and by the list
    for name, code in kernels:
        assert not _spills(code), name
        if "adapter_down_kernel" in name:
            assert _m0_is_the_transfers(code), name
            first = next(k for k, ln in enumerate(code) if "global_load_lds" in ln)
            last = max(k for k, ln in enumerate(code) if "v_mfma" in ln)
            assert not [ln for ln in code[first : last + 1] if re.search(r"global_load_(?!lds)|flat_load|buffer_load", ln)], name


def test_gated(tmp_path):
    kernels = list(_kernels(tmp_path, "gated.hip", "gated_\\w+_kernel|dense_few_kernel|dense_some_kernel"))
    assert len(kernels) == 2 * (5 + 6 + 5 + 5 + 1)  # some, few, pointwise and narrow of each activation; the bias's sums
    for name, code in kernels:
        assert not _spills(code), name
        if "dense_some" in name:
            assert _m0_is_the_transfers(code), name


def test_residual_norm(tmp_path):
    kernels = list(_kernels(tmp_path, "residual_norm.hip", "residual_norm_\\w*kernel"))
    assert len(kernels) == 3 * (6 + 1 + 3 * 2 * 3 + 4)
    for name, code in kernels:
        # 16-bit rows with both norms: 8 bytes of a shared gate's form, and rows of four pieces to a lane
        known = re.search(r"residual_norm_back_kernelILi[01]ELi(1ELb1ELi1|4ELb[01]ELi[12])E", name)
        assert not _spills(code) or known, name


def test_which_forms_of_the_residual_norm_spill(tmp_path):
    """16-bit rows: one piece to a lane with both norms and a shared gate; four pieces with a gate, but a row's own without the norm behind."""
    spilled = {m[0] for name, code in _kernels(tmp_path, "residual_norm.hip", "residual_norm_\\w*kernel") if _spills(code) and (m := re.search(r"ILi[012]ELi\dELb[01]ELi[012]E", name))}
    assert spilled <= {f"ILi{dt}ELi{rest}E" for dt in (0, 1) for rest in ("1ELb1ELi1", "4ELb1ELi1", "4ELb1ELi2", "4ELb0ELi1")}


def test_a_row_has_arrived_before_it_is_overwritten(tmp_path):
    """dx and dy may take the places of ds and y: without the norm behind, whose sums use both, a row's waves meet only when they have them, whatever else is on its way."""
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not build.Path(hipcc).exists():
        pytest.skip("needs hipcc")
    out = tmp_path / "kernels.s"
    res = subprocess.run([hipcc, *build.CXXFLAGS, *build.DEVICE_FLAGS, "-S", "--cuda-device-only", str(build.CSRC / "residual_norm.hip"), "-o", str(out)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
    lines, forms = out.read_text().split("\n"), 0
    for i, pieces in ((i, int(m[1])) for i, ln in enumerate(lines) if (m := re.match(r"^_ZN\S*residual_norm_back_kernelILi\dELi(\d)ELb0ELi\dE\S*: *;", ln))):
        body = lines[i : next(j for j in range(i, len(lines)) if lines[j].startswith(".Lfunc_end"))]
        meets = next(k for k, ln in enumerate(body) if "s_barrier" in ln and "lgkmcnt(0)" in body[k - 1] and "#ASM" in body[k - 2])
        used = [k for k, ln in enumerate(body[:meets]) if re.match(r"\s+; arrived v\[\d+:\d+\]", ln)]
        assert len(used) == 2 * pieces, lines[i]
        between = body[used[0] : meets]
        assert not [ln for ln in between if re.match(r"\s+(global|flat|buffer|scratch)_load", ln)], lines[i]
        forms += 1
    assert forms == 3 * 3 * 3
