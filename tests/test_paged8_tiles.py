"""CPU checks of how attention over pages of 8-bit values is divided: the numbers by which uncut
calls find their tiles (tests/cpp/paged_tiles_check.cpp), the pieces of cut ones
(tests/cpp/paged_units128_check.cpp)."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.mark.parametrize("name", ["paged_tiles_check", "paged_units128_check"])
def test_host_checks(tmp_path, name):
    exe = tmp_path / name
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Wno-unused-function", "-I", str(ROOT / "include"), "-I",
                    str(ROOT / "strict_amd" / "csrc"), str(ROOT / "tests" / "cpp" / f"{name}.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "failures=0" in r.stdout
