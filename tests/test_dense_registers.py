"""The dense kernels of few rows keep what they hold in registers: nothing in a call that memory or latency bounds goes to local memory (the compiler's report; no GPU)."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "denno_beta_b200", "csrc")


@pytest.mark.parametrize("four_bits", ["true", "false"])
def test_nothing_spills(four_bits, tmp_path):
    from denno_beta_b200 import build

    kinds = ["%s, %d, %d" % (four_bits, matrices, rows) for matrices in (1, 2) for rows in (16, 128)]
    source = tmp_path / "few.cu"
    source.write_text('#include "dense_tc.cuh"\n' + "".join("template __global__ void dnb::dt::dense_kernel<dnb::dt::Cfg<%s>>(const __grid_constant__ dnb::dt::Params);\n" % k for k in kinds))
    got = subprocess.run([build.NVCC, *build.FLAGS, "-Xptxas", "-v", "-cubin", str(source), "-o", str(tmp_path / "few.cubin")], capture_output=True, text=True)
    assert got.returncode == 0, got.stderr[-2000:]
    spills = re.findall(r"(\d+) bytes spill stores, (\d+) bytes spill loads", got.stderr + got.stdout)
    assert len(spills) == len(kinds) and set(spills) == {("0", "0")}, spills
