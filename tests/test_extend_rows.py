"""CPU checks of the way through a block's older rows (iq_extend_plan.h),
compiled with g++ and run here."""
import os
import subprocess
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))


def test_extend_rows():
    with tempfile.TemporaryDirectory() as d:
        exe = os.path.join(d, "test_extend_rows")
        subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=undefined", "-o", exe,
                        os.path.join(HERE, "cpp", "test_extend_rows.cpp")], check=True)
        r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "0 failures" in r.stdout and "runtime error" not in r.stderr, r.stderr
