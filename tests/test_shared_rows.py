"""The rows that the parts behind a shared prefix are joined for, on the host (tests/shared_rows.cpp)."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_rows_of_sequences(tmp_path):
    exe = str(tmp_path / "shared_rows")
    r = subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-o", exe, os.path.join(HERE, "shared_rows.cpp")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "rows of batches" in r.stdout
