"""What the compiler made of a serving step's kernels, read from the code objects that were built here."""
import os
import re
import subprocess

import pytest

BUILD = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "arcinferzero_amd", "csrc", "build")
LLVM = "/opt/rocm/llvm/bin"


@pytest.mark.parametrize("module", ["norm_rope", "plan", "attn_shared", "attn_shared_few", "sample"])
def test_memory_is_addressed_as_what_it_is(module, tmp_path):
    """Loads through pointers of no known address space wait for LDS and memory alike; packed f32 instructions are switched off for all kernels."""
    src, obj = os.path.join(BUILD, module + ".hsaco"), str(tmp_path / "o")
    if not os.path.exists(src) or not os.path.exists(os.path.join(LLVM, "llvm-objdump")):
        pytest.skip("the code objects are not built here")
    subprocess.run([os.path.join(LLVM, "clang-offload-bundler"), "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", "--input=" + src, "--output=" + obj, "--unbundle"], check=True)
    code = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", obj], capture_output=True, text=True, check=True).stdout
    assert len(re.findall(r"\bglobal_(load|store)_", code)) > 3
    assert not re.findall(r"\bflat_(load|store|atomic)\w*", code)
    assert not re.findall(r"\bv_pk_(add|mul|fma)_f32\b", code)
