"""Index rules of the int8 kernels that are plain C++, checked exhaustively on the CPU (tests/native/)."""

import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def run(tmp_path, name):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ is not available")
    exe = tmp_path / name
    subprocess.run([gxx, "-std=c++17", "-O2", "-Wall", "-Werror", "-o", str(exe),
                    str(ROOT / "tests" / "native" / f"{name}.cpp")], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout


def test_rows_read_only_their_columns(tmp_path):
    """Rows that start anywhere are read in 16-byte granules; padding between rows is not read."""
    assert "OK 34560 layouts" in run(tmp_path, "int8_span_check")


def test_pair_schedule(tmp_path):
    """Tiles, splits and slots of the CTA-pair kernel: every k-block once, waits only on pairs dispatched before."""
    out = run(tmp_path, "int8_sched_check")
    assert out.startswith("OK ") and "schedules" in out
