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


def _tensors():
    g = torch.Generator(device="cuda").manual_seed(70)
    a = torch.randint(-9, 9, (8, 32), generator=g, device="cuda", dtype=torch.int8)
    return dict(a=a, b=a[:6], e=a[:6].repeat(3, 1).view(3, 6, 32), x=torch.randn(2, 9, 32, device="cuda"),
                v=torch.ones(6, device="cuda"),
                offsets=torch.tensor([0, 2, 4, 8], dtype=torch.int32, device="cuda"),
                index=torch.zeros(5, dtype=torch.int32, device="cuda"))


REFUSED = {
    "a wider than b": lambda t: m.matmul(t["a"][:, :16], t["b"]),
    "a on the CPU": lambda t: m.matmul(t["a"].cpu(), t["b"]),
    "b on the CPU": lambda t: m.matmul(t["a"], t["b"].cpu()),
    "a in floats": lambda t: m.matmul(t["a"].float(), t["b"]),
    "a off its alignment": lambda t: m.matmul(t["a"].view(-1)[1:225].view(7, 32), t["b"]),
    "a of an odd pitch": lambda t: m.matmul(t["a"].view(-1)[:132].view(6, 22), t["b"][:, :22]),
    "a transposed": lambda t: m.matmul(t["a"].t(), t["b"][:, :8]),
    "a with overlapping rows": lambda t: m.matmul(t["a"].as_strided((4, 32), (16, 1)), t["b"]),
    "a of three dimensions": lambda t: m.matmul(t["a"][None], t["b"]),
    "k of nothing": lambda t: m.matmul(t["a"][:, :0], t["b"][:, :0]),
    "float64 result": lambda t: m.matmul(t["a"], t["b"], dtype=torch.float64),
    "int32 result": lambda t: m.matmul(t["a"], t["b"], dtype=torch.int32),
    "int8 without a step": lambda t: m.matmul(t["a"], t["b"], dtype=torch.int8),
    "a step without int8": lambda t: m.matmul(t["a"], t["b"], out_scale=1.0),
    "a step of zero": lambda t: m.matmul(t["a"], t["b"], dtype=torch.int8, out_scale=0.0),
    "a step beyond fp32": lambda t: m.matmul(t["a"], t["b"], dtype=torch.int8, out_scale=1e300),
    "a short bias": lambda t: m.matmul(t["a"], t["b"], bias=t["v"][:5]),
    "a bias in bf16": lambda t: m.matmul(t["a"], t["b"], bias=t["v"].bfloat16()),
    "a strided bias": lambda t: m.matmul(t["a"], t["b"], bias=t["v"].repeat(2)[::2]),
    "a bias on the CPU": lambda t: m.matmul(t["a"], t["b"], bias=t["v"].cpu()),
    "a residual of another type": lambda t: m.matmul(t["a"], t["b"], dtype=torch.float16,
                                                     residual=torch.zeros(8, 6, device="cuda")),
    "a broadcast residual": lambda t: m.matmul(t["a"], t["b"], residual=torch.zeros(
        1, 6, device="cuda").expand(8, 6)),
    "an int8 residual": lambda t: m.matmul(t["a"], t["b"], out_scale=1.0, residual=torch.zeros(
        8, 6, device="cuda", dtype=torch.int8)),
    "an unknown activation": lambda t: m.matmul(t["a"], t["b"], activation="tanh"),
    "experts of two dimensions": lambda t: m.grouped_matmul(t["a"], t["b"], t["offsets"]),
    "short offsets": lambda t: m.grouped_matmul(t["a"], t["e"], t["offsets"][:3]),
    "offsets of 64 bits": lambda t: m.grouped_matmul(t["a"], t["e"], t["offsets"].long()),
    "no offsets": lambda t: m.grouped_matmul(t["a"], t["e"], None),
    "one bias for all experts": lambda t: m.grouped_matmul(t["a"], t["e"], t["offsets"], bias=t["v"]),
    "overlapping experts": lambda t: m.grouped_matmul(t["a"], t["e"].as_strided((3, 6, 32), (32, 32, 1)),
                                                      t["offsets"]),
    "integers to quantise": lambda t: m.quantize_rows(t["a"]),
    "rows of nothing": lambda t: m.quantize_rows(t["x"][0][:, :0]),
    "an index of 64 bits": lambda t: m.quantize_rows(t["x"][0], t["index"].long()),
    "a strided index": lambda t: m.quantize_rows(t["x"][0], t["index"][::2]),
    "columns apart": lambda t: m.quantize_rows(t["x"][0].t()),
    "a vector to quantise": lambda t: m.quantize_rows(t["v"]),
    "groups that do not divide": lambda t: m.group_norm(t["x"], 5),
    "no groups": lambda t: m.group_norm(t["x"], 0),
    "groups beyond 32 bits": lambda t: m.group_norm(t["x"], 1 << 40),
    "eps below zero": lambda t: m.group_norm(t["x"], 4, eps=-1.0),
    "eps beyond fp32": lambda t: m.group_norm(t["x"], 4, eps=1e300),
    "float64 to normalise": lambda t: m.group_norm(t["x"].double(), 4),
    "channels apart": lambda t: m.group_norm(t["x"].transpose(1, 2), 3),
    "uneven positions": lambda t: m.group_norm(t["x"].repeat(1, 2, 1)[:, :9], 4),
    "a short gamma": lambda t: m.group_norm(t["x"], 4, torch.ones(31, device="cuda")),
    "a beta on the CPU": lambda t: m.group_norm(t["x"], 4, None, torch.ones(32)),
    "int8 norm without a step": lambda t: m.group_norm(t["x"], 4, dtype=torch.int8),
    "too many channels": lambda t: m.group_norm(torch.zeros(1, 2, 8200, device="cuda"), 1),
}


@pytest.mark.parametrize("what", REFUSED)
def test_compiled_and_checked_calls_refuse_alike(cuda, what, monkeypatch):
    operators._load_torch()
    assert operators._calls is not None, "torch_calls.so was not built"
    t = _tensors()
    before = m.launch_count()
    with pytest.raises((ValueError, m.Int8ConvError)) as compiled:
        REFUSED[what](t)
    monkeypatch.setattr(operators, "_calls", None)
    with pytest.raises((ValueError, m.Int8ConvError)) as checked:
        REFUSED[what](t)
    assert m.launch_count() == before
    assert type(compiled.value) is type(checked.value) and str(compiled.value) == str(checked.value)


def test_channels_beyond_32_bits(cuda):
    operators._load_torch()
    x = torch.empty(1, 1, (1 << 32) + 32, dtype=torch.bfloat16, device="cuda")
    before = m.launch_count()
    with pytest.raises(ValueError, match="range"):
        m.group_norm(x, 4)
    assert m.launch_count() == before


def test_results_carry_no_gradients(cuda):
    # Trainable inputs are taken as values, and left as they are.
    t = _tensors()
    gamma = torch.nn.Parameter(torch.ones(32, device="cuda"))
    x = t["x"].clone().requires_grad_()
    bias = torch.nn.Parameter(t["v"])
    y = m.group_norm(x, 4, gamma)
    z = m.matmul(t["a"], t["b"], bias=bias)
    q, scale = m.quantize_rows(x[0])
    for r in (y, z, q, scale):
        assert not r.requires_grad and r.grad_fn is None
    assert torch.equal(y, m.group_norm(t["x"], 4)) and x.grad is None and gamma.grad is None
