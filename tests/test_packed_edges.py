"""Packed-batch operators at the edges of what their entries take, without a GPU."""
import concurrent.futures
import math
import re
import subprocess

import pytest
import torch

from torchft_b200 import _build
from torchft_b200.ops import kernels as K


def test_the_masked_attention_kernels_keep_nothing_in_local_memory(tmp_path):
    """Their warpgroups share out registers, and no value of one share lies where another looks for it: the compiler's own report."""

    def report(name):
        src = _build.CSRC / "kernels" / f"{name}.cu"
        cmd = [_build._nvcc(), *_build.NVCC_FLAGS, f"-I{_build.CSRC / 'kernels'}", "-Xptxas", "-v", "-c", str(src), "-o", str(tmp_path / f"{name}.o")]
        proc = subprocess.run(cmd, capture_output=True, text=True)
        assert proc.returncode == 0, proc.stderr
        return re.findall(r"Compiling entry function '(\S+)'.*?(\d+) bytes stack frame, (\d+) bytes spill stores, (\d+) bytes spill loads",
                          proc.stdout + proc.stderr, re.S)

    with concurrent.futures.ThreadPoolExecutor(2) as pool:
        fwd, bwd = pool.map(report, ("attention_masked_fwd_tcgen05", "attention_bwd_tcgen05"))
    assert len(fwd) == 4
    masked = fwd + [r for r in bwd if "ELb1E" in r[0]]
    assert len(masked) == 8
    assert all(r[1:] == ("0", "0", "0") for r in masked), masked
