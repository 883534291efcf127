"""Which pieces of rows of 8-bit integers the kernels load, on the CPU (tests/cpp/i8_rows_check.cpp)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rows_are_loaded_to_their_end_and_no_further(tmp_path):
    exe = str(tmp_path / "i8_rows_check")
    subprocess.check_call(["g++", "-std=c++17", "-O1", os.path.join(ROOT, "tests", "cpp", "i8_rows_check.cpp"), "-o", exe])
    out = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stdout + out.stderr
