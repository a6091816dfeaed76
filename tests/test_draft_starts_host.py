"""Ranges of packed nodes from starts of any value, on the host (tests/native/node_range_check.cpp)."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.skipif(shutil.which("hipcc") is None, reason="hipcc not on PATH")
def test_ranges_of_any_starts(tmp_path):
    exe = tmp_path / "node_range_check"
    subprocess.run(["hipcc", "-std=c++17", "-O2", f"-I{ROOT / 'ds4cuda_amd' / 'csrc'}",
                    str(ROOT / "tests" / "native" / "node_range_check.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and " 0 wrong" in out.stdout, out.stdout + out.stderr
