"""What the block-scaled product's kernels rely on in the generated code: M0, which the loads to LDS take their target from
in inline assembly without the compiler knowing, is used by nothing else."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCES = ["och_gemm_f8_few_44.hip", "och_gemm_f8_pipe_45.hip"]


@pytest.mark.parametrize("source", SOURCES)
def test_m0_is_used_by_the_loads_to_lds_only(source, tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc is not available")
    out = str(tmp_path / "k.s")
    subprocess.run([hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-ffp-contract=off", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                    "-Wno-unused-command-line-argument", "--cuda-device-only", "-S", os.path.join(ROOT, "ocean-tensor-package_amd", "csrc", source), "-o", out],
                   check=True, capture_output=True)
    lines = [ln.split(";")[0].strip() for ln in open(out)]
    code = [ln for ln in lines if ln and not ln.startswith(".") and not ln.endswith(":")]
    uses = [i for i, ln in enumerate(code) if re.search(r"\bm0\b", ln)]
    assert len(uses) >= 8, "no load to LDS found in %s" % source
    for i in uses:
        assert re.fullmatch(r"s_mov_b32 m0, s\d+", code[i]), code[i]
        assert any(c.startswith("global_load_lds_dword") for c in code[i + 1:i + 3]), code[i:i + 3]
