"""kv_evict's selection and its lists of moves on the host: the kernel's own
arithmetic against a sort, with NaN weights on both sides of the places left,
protected slots, ties, weights of every size, and rows off the batch size."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def test_selection_equals_a_sort(tmp_path):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no host compiler")
    program = tmp_path / "evict_select"
    subprocess.run([compiler, "-O2", "-std=c++17", "-Wall", "-Wextra", "-Werror", f"-I{ROOT / 'cruise_amd' / 'csrc'}",
                    str(ROOT / "tests" / "native" / "evict_select.cpp"), "-o", str(program)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout
