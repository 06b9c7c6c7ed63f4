"""The paged key-value cache at its edges, without a GPU."""
import os
import subprocess

from fbgemm_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rules_at_the_edges(tmp_path):
    exe = str(tmp_path / "paged_edges_test")
    cuda = os.path.join(os.path.dirname(os.path.dirname(build._nvcc())), "include")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", build.CSRC, "-I", build.INCLUDE, "-I", cuda,
                    os.path.join(ROOT, "tests", "cpp", "paged_edges_test.cc"), "-o", exe], check=True)
    res = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0, res.stdout
