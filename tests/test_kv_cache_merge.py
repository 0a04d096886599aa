"""Code generation of the 4-bit decode's merge kernel (CPU: hipcc cross-compiles
csrc/kv_decode_merge.hip for gfx950 to assembly): no scratch."""

import os
import shutil
import subprocess

import pytest

from test_kv_cache_codegen import CSRC, HIPCC, ROOT, kernels


@pytest.mark.skipif(not shutil.which(HIPCC), reason="hipcc not available")
def test_no_scratch(tmp_path):
    out = tmp_path / "merge.s"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang",
                    "-target-feature", "-Xclang", "-packed-fp32-ops", "--cuda-device-only", "-S",
                    f"-I{os.path.join(ROOT, 'include')}", f"-I{CSRC}",
                    os.path.join(CSRC, "kv_decode_merge.hip"), "-o", str(out)], check=True,
                   capture_output=True)
    found = kernels(out.read_text())
    assert len(found) == 1
    for name, (regs, scratch, code) in found.items():
        assert "kv_decode_merge_kernel" in name
        assert scratch == 0 and "scratch_" not in code and regs <= 64
