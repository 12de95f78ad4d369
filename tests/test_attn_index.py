"""The rows, pages and positions that the attention block's kernels work out of a batch in device memory, on the host: nothing that the
batch says, however wrong, leads out of a buffer (tests/attn_index.cpp, with the compiler's checks for overflow)."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_places_stay_in_their_buffers(tmp_path):
    exe = str(tmp_path / "attn_index")
    r = subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-o", exe, os.path.join(HERE, "attn_index.cpp")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "in their buffers" in r.stdout
