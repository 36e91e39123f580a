"""The page accounting of the native runtime, from a program of its own (no GPU)."""
import os
import subprocess

from safetyraise_lmengine_b200.csrc import build

HERE = os.path.dirname(os.path.abspath(__file__))


def test_calls_that_run_out_of_memory_change_nothing(tmp_path):
    host = os.path.join(build.HERE, "host")
    program = str(tmp_path / "pages")
    sources = [os.path.join(host, f) for f in sorted(os.listdir(host)) if f.endswith(".cpp")]
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", host, os.path.join(HERE, "native", "pages_out_of_memory.cpp"), *sources, "-o", program],
                   check=True)
    r = subprocess.run([program], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr
