"""Rows and keys of sequences behind a shared prefix, on the host: the two parts of an interval are the whole of it, and inside the buffers whatever these
hold (tests/shared_index.cpp, with the compiler's checks for overflow)."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_parts_of_intervals(tmp_path):
    exe = str(tmp_path / "shared_index")
    r = subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-o", exe, os.path.join(HERE, "shared_index.cpp")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "places of shared prefixes" in r.stdout
