"""The operators' compiled calls: what they do with a launch that fails, and that
they refuse what the checks in Python refuse."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import int8_kernel_lab_b200 as m
from int8_kernel_lab_b200 import operators

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


def test_failed_launch_is_not_tried_again(cuda):
    # A capture that something else has broken lets no launch through: an error
    # on the host, before the GPU sees anything.  y += a @ b.T must not be tried twice.
    code = """
import torch, int8_kernel_lab_b200 as m
from int8_kernel_lab_b200 import operators
a = torch.ones(40, 64, dtype=torch.int8, device="cuda")
x = torch.randn(2, 20, 64, device="cuda")
y = torch.zeros(40, 40, device="cuda")
off = torch.tensor([0, 10, 40], dtype=torch.int32, device="cuda")
q, s = torch.empty_like(a), torch.empty(40, device="cuda")
m.launch_matmul(a, a, y, residual=y)
assert operators._calls is not None
g = torch.cuda.CUDAGraph()
stream = torch.cuda.Stream()
torch.cuda.synchronize()
with torch.cuda.stream(stream):
    g.capture_begin()
    try:
        torch.cuda.synchronize()
    except Exception:
        pass
    for call in (lambda: m.launch_matmul(a, a, y, residual=y),
                 lambda: m.launch_grouped_matmul(a, a.view(1, 40, 64), off[:2], y),
                 lambda: m.launch_quantize_rows(x.view(40, 64), q, s)):
        before = m.launch_count()
        try:
            call()
        except m.Int8ConvError as e:
            print("status", e)
        else:
            raise SystemExit("a launch into a broken capture went through")
        assert m.launch_count() == before + 1, m.launch_count() - before
print("done")
import os, sys
sys.stdout.flush()
os._exit(0)   # the broken capture is left as it is
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True,
                          timeout=120)
    assert done.returncode == 0 and "done" in done.stdout, done.stdout + done.stderr[-2000:]
