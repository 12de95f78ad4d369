"""Plans of sequences whose first pages others share, on the host: no row in a shared page, no page lost (tests/plan_shared.cpp)."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_pages_of_others_get_no_rows(tmp_path):
    exe = str(tmp_path / "plan_shared")
    r = subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-o", exe, os.path.join(HERE, "plan_shared.cpp")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "places of plans behind prefixes" in r.stdout
