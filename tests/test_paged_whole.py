"""CPU check of the division of an attention call whose tiles are not cut
(tests/cpp/paged_whole_check.cpp)."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_every_tile_is_one_workers(tmp_path):
    exe = tmp_path / "paged_whole_check"
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Wno-unused-function", "-I", str(ROOT / "include"), "-I",
                    str(ROOT / "strict_amd" / "csrc"), str(ROOT / "tests" / "cpp" / "paged_whole_check.cpp"), "-o", str(exe)],
                   check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "failures=0" in r.stdout
