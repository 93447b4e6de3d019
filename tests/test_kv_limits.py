"""The cache's host bookkeeping and argument checks at the ends of their ranges, on the CPU (tests/kv_limits_host.cpp)."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
CXX = shutil.which("c++") or shutil.which("g++")


def test_limits(tmp_path):
    if CXX is None:
        pytest.skip("no C++ compiler")
    out = tmp_path / "kv_limits_host"
    r = subprocess.run([CXX, "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-I", str(ROOT / "include"),
                        str(ROOT / "tests" / "kv_limits_host.cpp"), "-o", str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([str(out)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "kv limits ok" in r.stdout, r.stdout + r.stderr
