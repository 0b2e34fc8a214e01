"""CPU checks of the split that the attention kernels make (iq_attn_plan.h),
compiled with g++ and run here: chunks by a reciprocal that is as far off as it
may be, and the choice of a chunk's size."""
import os
import subprocess
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))


def test_attention_split():
    with tempfile.TemporaryDirectory() as d:
        exe = os.path.join(d, "test_attn_split")
        subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-fsanitize=undefined", "-o", exe,
                        os.path.join(HERE, "cpp", "test_attn_split.cpp")], check=True)
        r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "0 failures" in r.stdout and "runtime error" not in r.stderr, r.stdout + r.stderr
