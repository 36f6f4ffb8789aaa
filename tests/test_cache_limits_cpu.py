"""The sequence-cache operators at their limits, without a GPU: that no address
leaves its array whatever device memory holds."""
import os
import subprocess

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_addresses_stay_inside(tmp_path):
    exe = tmp_path / "paged_bounds_check"
    r = subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-fsanitize=undefined",
                        "-fno-sanitize-recover=all", "-I", os.path.join(REPO, "kernel.h_amd", "csrc", "kernels"),
                        os.path.join(REPO, "tests", "cpp", "paged_bounds_check.cpp"), "-o", str(exe)],
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert r.returncode == 0, r.stdout
    r = subprocess.run([str(exe)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip().endswith("paged_bounds_check ok"), r.stdout
