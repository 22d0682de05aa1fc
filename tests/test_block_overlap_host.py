"""Which strided tensors share bytes: csrc/tde_overlap.h against sets of bytes, compiled for the host."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_regions_against_sets_of_bytes(tmp_path):
    program = str(tmp_path / "unit_test_overlap")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "torch_dist_ext_amd", "csrc"),
                    os.path.join(ROOT, "tests", "native", "unit_test_overlap.cpp"), "-o", program], check=True, timeout=300)
    ran = subprocess.run([program], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert ran.returncode == 0, ran.stdout
