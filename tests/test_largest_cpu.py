"""The search for a row's largest classes, run on the CPU at the borders of what a group of waves holds (tests/cpp/largest_check.cpp)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CLANG = "/opt/rocm/lib/llvm/bin/clang++"   # the stand-in for the device's header needs a compiler that has its vector types


@pytest.mark.skipif(not os.path.exists(CLANG), reason="needs ROCm's clang++")
def test_the_search_for_the_largest_ends_with_them(tmp_path):
    exe, cpp = str(tmp_path / "largest_check"), os.path.join(ROOT, "tests", "cpp")
    subprocess.check_call([CLANG, "-x", "c++", "-std=c++17", "-O2", "-w", "-I" + os.path.join(cpp, "host_kernels"), os.path.join(cpp, "largest_check.cpp"), "-o", exe])
    out = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr
