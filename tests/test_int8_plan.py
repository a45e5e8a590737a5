"""The plans of int8_linear on the host: no workgroup has more channels than its
kernel computes, over every inner size and the channels that are cut into ranges."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def test_every_channel_has_a_tile(tmp_path):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no host compiler")
    program = tmp_path / "int8_plan"
    subprocess.run([compiler, "-O2", "-std=c++17", "-Wall", "-Wextra", "-Werror", f"-I{ROOT / 'cruise_amd' / 'csrc'}",
                    str(ROOT / "tests" / "native" / "int8_plan.cpp"), "-o", str(program)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout


def test_every_plan_has_a_kernel(tmp_path):
    """Plans without a kernel are told apart (they end a call with an error), and no sizes lead to one."""
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no host compiler")
    program = tmp_path / "int8_kernels"
    subprocess.run([compiler, "-O2", "-std=c++17", "-Wall", "-Wextra", "-Werror", f"-I{ROOT / 'cruise_amd' / 'csrc'}",
                    str(ROOT / "tests" / "native" / "int8_kernels.cpp"), "-o", str(program)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout
