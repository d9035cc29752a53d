"""Registers of linear_cross_entropy's kernels: 11 warps share the register file, and the forward's epilogue holds 128 accumulators a
thread.  The compiler's own report, no GPU."""
import os
import re
import shutil
import subprocess

import pytest

from streamep_b200 import _ext

NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"


@pytest.mark.skipif(not os.path.exists(NVCC), reason="no CUDA compiler")
def test_nothing_spills(tmp_path):
    out = subprocess.run([NVCC, *_ext.NVCC_FLAGS, "-Xptxas", "-v", "-cubin", "-o", str(tmp_path / "x.cubin"), str(_ext._CSRC / "linear_loss_kernels.cu")],
                         capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stderr[-2000:]
    report = re.findall(r"Compiling entry function '(\w*linear_loss_kernelILb\w*)'.*?(\d+) bytes spill stores, (\d+) bytes spill loads.*?Used (\d+) registers", out.stderr, re.S)
    assert len({m for m, *_ in report}) == 4, out.stderr[-2000:]       # forward and backward, tokens as rows and as columns
    for name, stores, loads, registers in report:
        assert (int(stores), int(loads)) == (0, 0) and int(registers) <= 168, (name, stores, loads, registers)
