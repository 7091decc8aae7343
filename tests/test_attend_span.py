"""Which tokens attention looks up in a block table: none past the table's last column, whatever the
window and the context, and every one that a row sees (``tests/attend_span_check.cpp``)."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

SRC = Path(__file__).with_name("attend_span_check.cpp")


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_every_lookup_lies_in_the_table(tmp_path):
    exe = tmp_path / "span"
    subprocess.run(["g++", "-O2", "-std=c++17", "-o", str(exe), str(SRC)], check=True, capture_output=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr
