"""The C++ host surface of the 8-bit operators, the routing and the experts (include/miaie.hpp)
over recording entry points: no library, no GPU (tests/host_experts_check.cpp)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_wrappers_refuse_what_does_not_fit(tmp_path):
    exe = str(tmp_path / "host_experts_check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Wextra", "-Werror", f"-I{os.path.join(ROOT, 'include')}",
                    os.path.join(ROOT, "tests", "host_experts_check.cpp"), "-o", exe], check=True, timeout=300)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
