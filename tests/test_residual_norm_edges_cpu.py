"""fw_residual_norm's host side without a GPU: argument values that the header allows must reach the launch, whatever they are."""
import os
import subprocess
import sys

import pytest
import torch

from conftest import ROOT

CALL = """
import ctypes
from fantasy_world_amd import hip_ops
lib = hip_ops.load_library()
x, y, h, bias = (ctypes.c_void_p(i << 44) for i in (1, 2, 3, 4))            # addresses that nothing reads: the call ends at the launch
rc = lib.fw_residual_norm(x, 256, x, 256, 2, y, 256, 1, bias, None, None, 0, None, 1, None, None, None, None, ctypes.c_float(1e-6), h, 256, 1, None, {rows}, 256, {rpm}, None)
print("returned", rc)
"""


@pytest.mark.skipif(torch.cuda.is_available(), reason="the call stops at the launch only where there is no GPU")
@pytest.mark.parametrize("rows,rpm", [(4096, 0x7fffffff), (4096, 0x7fffffff - 4094), (5000, 0x7fffffff - 3000), (0x7fffffff, 0x7fffffff), (0x7fffffff, 0x40000000)])
def test_one_vector_for_all_rows(rows, rpm):
    """rows_per_mod >= rows is how a caller says it; the number of runs is then 1 for every value up to the largest int."""
    r = subprocess.run([sys.executable, "-c", CALL.format(rows=rows, rpm=rpm)], cwd=ROOT, capture_output=True, text=True, timeout=120, env=dict(os.environ, PYTHONPATH=ROOT))
    assert r.returncode == 0 and "returned" in r.stdout and "returned -1" not in r.stdout, (r.returncode, r.stdout, r.stderr[-500:])
