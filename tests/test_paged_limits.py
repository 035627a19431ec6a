"""CPU checks of the paged operators: argument checks at their largest sizes
(tests/cpp/paged_limits_check.cpp), the division of a call by the tiles, units and pieces
that the kernels take (tests/cpp/paged_units_check.cpp)."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.mark.parametrize("name", ["paged_limits_check", "paged_units_check"])
def test_host_checks(tmp_path, name):
    exe = tmp_path / name
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Wno-unused-function", "-I", str(ROOT / "include"), "-I",
                    str(ROOT / "strict_amd" / "csrc"), str(ROOT / "tests" / "cpp" / f"{name}.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "failures=0" in r.stdout
