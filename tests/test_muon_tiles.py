"""What shares a workgroup's LDS in the Newton-Schulz products, on the CPU."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def test_no_strip_reaches_another_waves_sums(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    exe = tmp_path / "muon_tiles"
    subprocess.run([cxx, "-std=c++17", "-Wall", str(ROOT / "tests" / "muon_tiles.cpp"), "-o", str(exe)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0, res.stdout
