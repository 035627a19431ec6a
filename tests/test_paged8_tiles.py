"""CPU check of the numbers by which uncut calls over pages of 8-bit values find their tiles
(tests/cpp/paged_tiles_check.cpp)."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_find_tile(tmp_path):
    exe = tmp_path / "paged_tiles_check"
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-I", str(ROOT / "include"), "-I", str(ROOT / "strict_amd" / "csrc"),
                    str(ROOT / "tests" / "cpp" / "paged_tiles_check.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "failures=0" in r.stdout
