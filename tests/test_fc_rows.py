"""CPU test of the addresses of rows in tensors of very many columns (csrc/fc_mma.cuh), compiled for the host: no step between rows is formed in 32 bits."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_steps_between_rows(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("nvcc not found")
    exe = str(tmp_path / "fc_rows_check")
    src = os.path.join(ROOT, "tests", "fc_rows_check.cu")
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O1", "-std=c++17", "-Xcompiler", "-fwrapv", "-o", exe, src], check=True, capture_output=True, timeout=300)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stdout + out.stderr


def test_all_steps_are_formed_so():
    text = open(os.path.join(ROOT, "dragon-alpha-v1.0_b200", "csrc", "fc_mma.cuh")).read()
    steps = re.findall(r"\b(?:to|from) \+= ([^)\n]*\)?)", text)
    assert len(steps) == 2 and all(s.startswith("fc_rows_on(") for s in steps), steps
