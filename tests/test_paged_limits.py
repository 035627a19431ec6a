"""CPU checks of the paged operators at their largest sizes (tests/cpp/paged_limits_check.cpp)."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_largest_sizes(tmp_path):
    exe = tmp_path / "paged_limits_check"
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-I", str(ROOT / "include"), "-I",
                    str(ROOT / "strict_amd" / "csrc"), str(ROOT / "tests" / "cpp" / "paged_limits_check.cpp"),
                    "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "failures=0" in r.stdout
