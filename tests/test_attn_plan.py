"""CPU checks of infer_amd/csrc/iq_attn_plan.h, compiled with g++ and run
here: a token's page for every page size, and that the split of a batch over
workgroups covers every token, leaves no chunk empty and stays within the
grid and the partial results that the host plans for."""
import os
import subprocess
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))


def test_attention_plans():
    with tempfile.TemporaryDirectory() as d:
        exe = os.path.join(d, "test_attn_plan")
        subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-o", exe, os.path.join(HERE, "cpp", "test_attn_plan.cpp")],
                       check=True)
        r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "0 failures" in r.stdout
