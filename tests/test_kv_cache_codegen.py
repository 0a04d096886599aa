"""Code-generation checks of the cache operators' kernels (CPU: hipcc
cross-compiles csrc/kv_append.hip and csrc/kv_decode.hip for gfx950 to
assembly).

A kernel that uses scratch pays for it at every launch (the 4-bit decode of a
short request took 17 us for 10 with a few spilled registers), and the decode
counts on two waves a SIMD, the appends on six; block ids have to be scalar
loads and tiles buffer loads (no address arithmetic in vector registers)."""

import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "mla-decode-kernels_amd", "csrc")
HIPCC = "/opt/rocm/bin/hipcc"

pytestmark = pytest.mark.skipif(not shutil.which(HIPCC), reason="hipcc not available")


@pytest.fixture(scope="module", params=["kv_append", "kv_decode"])
def asm(request, tmp_path_factory):
    out = tmp_path_factory.mktemp("kv_asm") / f"{request.param}.s"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang",
                    "-target-feature", "-Xclang", "-packed-fp32-ops", "--cuda-device-only", "-S",
                    f"-I{os.path.join(ROOT, 'include')}", f"-I{CSRC}",
                    os.path.join(CSRC, f"{request.param}.hip"), "-o", str(out)], check=True,
                   capture_output=True)
    return request.param, out.read_text()


def kernels(text):
    """{name: (registers, scratch bytes, code)} of every kernel."""
    out = {}
    for m in re.finditer(r"^(_Z\w+):.*?\n(.*?)^\.Lfunc_end.*?; TotalNumVgprs: (\d+).*?"
                         r"; ScratchSize: (\d+)", text, re.S | re.M):
        out[m.group(1)] = (int(m.group(3)), int(m.group(4)), m.group(2))
    return out


def test_no_scratch_and_enough_waves(asm):
    name, text = asm
    found = kernels(text)
    assert len(found) == {"kv_append": 7, "kv_decode": 3}[name]
    for kernel, (regs, scratch, code) in found.items():
        assert scratch == 0 and "scratch_" not in code, kernel
        limit = 256 if "kv_decode_kernel" in kernel else 80
        assert regs <= limit, (kernel, regs)


def test_decode_reads_tiles_through_buffers(asm):
    name, text = asm
    if name != "kv_decode":
        pytest.skip("the decode kernels only")
    for kernel, (_, _, code) in kernels(text).items():
        if "kv_decode_kernel" not in kernel:
            continue
        loop = code[code.index("v_mfma_scale"):]
        assert "buffer_load_dwordx4" in loop and "s_load_dword" in loop, kernel
        # No packed fp32 arithmetic.
        assert not re.search(r"v_pk_(add|mul|fma)_f32", code), kernel
