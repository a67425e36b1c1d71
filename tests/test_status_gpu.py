"""The device status is read from the units that have launched something.  Needs a B200."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = """
import torch
from torch.profiler import ProfilerActivity, profile
import ozaki_triton_b200 as oz

def copies():
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        assert oz.device_status() == 0
    return sum(e.count for e in p.key_averages() if "DtoH" in e.key)

copies()                                                # the profiler's own start
found = [copies()]
a = torch.randn(64, 64, device="cuda", dtype=torch.float64)
oz.ozaki_matmul(a, a)
found.append(copies())
oz.orthogonalize(torch.randn(300, 400, device="cuda"))
found.append(copies())
x, w = torch.ones(4, 64, device="cuda").half(), torch.ones(1, 64, 64, device="cuda").half()
oz.grouped_matmul(x, w, torch.tensor([0, 4], device="cuda"))
found.append(copies())
print("copies", *found)
"""


def test_only_units_with_launches_are_read():
    out = subprocess.run([sys.executable, "-c", SCRIPT], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    # nothing yet; the split and the cross GEMM; and a word for each further unit
    assert out.stdout.strip().splitlines()[-1] == "copies 0 2 3 4"
