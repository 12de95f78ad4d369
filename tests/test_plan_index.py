"""What a plan makes of a sequence's length and pages, on the host: right against 64-bit arithmetic, and inside the table whatever the
buffers hold (tests/plan_index.cpp, with the compiler's checks for overflow)."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_changes_of_sequences(tmp_path):
    exe = str(tmp_path / "plan_index")
    r = subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-o", exe, os.path.join(HERE, "plan_index.cpp")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "places of plans" in r.stdout
