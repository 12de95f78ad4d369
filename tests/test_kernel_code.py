"""What the compiler made of the kernels, read from the code objects that were built here."""
import os
import re
import subprocess

import pytest

BUILD = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "arcinferzero_amd", "csrc", "build")
LLVM = "/opt/rocm/llvm/bin"


@pytest.mark.parametrize("module", ["rope", "kv", "attn_few", "attn_many"])
def test_global_memory_is_addressed_as_such(module, tmp_path):
    """A load through a pointer of no known address space (flat_load) counts among the LDS reads and returns out of order: every wait for an
    operand from LDS behind it is one for memory."""
    src, obj = os.path.join(BUILD, module + ".hsaco"), str(tmp_path / "o")
    if not os.path.exists(src) or not os.path.exists(os.path.join(LLVM, "llvm-objdump")):
        pytest.skip("the code objects are not built here")
    subprocess.run([os.path.join(LLVM, "clang-offload-bundler"), "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", "--input=" + src, "--output=" + obj, "--unbundle"], check=True)
    code = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", obj], capture_output=True, text=True, check=True).stdout
    assert len(re.findall(r"\bglobal_(load|store)_", code)) > 3
    assert not re.findall(r"\bflat_(load|store|atomic)\w*", code)
