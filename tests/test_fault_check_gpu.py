"""What a fault check costs: one read of one word, whichever kernels have run in the process."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import time, torch
from vibecheck_nn_b200 import _lib, linear

def cost():
    best = 1e9
    for _ in range(300):
        t = time.perf_counter()
        _lib.fault_check()
        best = min(best, time.perf_counter() - t)
    return best

torch.zeros(1, device='cuda')
before = cost()
for dtype in (torch.float32, torch.bfloat16, torch.float16):
    x = torch.ones(512, 512, device='cuda', dtype=dtype)
    linear.linear_forward(x, x)
torch.cuda.synchronize()
print(before, cost())
"""


def test_fault_check_costs_the_same_after_a_linear_layer():
    """The shortest of 300 checks on either side, in a process of its own; two more copies and
    waits would make it some three times as long."""
    out = subprocess.run([sys.executable, '-c', PROGRAM], capture_output=True, text=True, timeout=300,
                         cwd=ROOT)
    assert out.returncode == 0, out.stderr[-2000:]
    before, after = map(float, out.stdout.split())
    assert after <= 1.5 * before, (before, after)
