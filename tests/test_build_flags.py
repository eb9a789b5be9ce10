"""CPU: the library's own code objects hold no packed fp32 instruction (the Makefile says why)."""
import glob
import os
import re
import subprocess

import pytest

BUILD = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lira-ann-search_amd", "build")
LLVM = "/opt/rocm/llvm/bin/"
OBJECTS = sorted(glob.glob(os.path.join(BUILD, "lira_*.o")))


@pytest.mark.skipif(not OBJECTS or not os.path.exists(LLVM + "llvm-objdump"), reason="needs the objects of a build, and LLVM's tools")
@pytest.mark.parametrize("obj", OBJECTS, ids=os.path.basename)
def test_no_packed_fp32(obj, tmp_path):
    bundle, code = str(tmp_path / "bundle"), str(tmp_path / "code")
    subprocess.run([LLVM + "llvm-objcopy", "--dump-section=.hip_fatbin=" + bundle, obj, os.devnull], check=True)
    subprocess.run([LLVM + "clang-offload-bundler", "--type=o", "--unbundle", "--input=" + bundle,
                    "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", "--output=" + code], check=True)
    text = subprocess.run([LLVM + "llvm-objdump", "-d", code], check=True, capture_output=True, text=True).stdout
    assert "s_endpgm" in text or "lira_merge" in obj or "lira_abi" in obj
    assert not re.search(r"v_pk_(add|mul|fma)_f32", text)
