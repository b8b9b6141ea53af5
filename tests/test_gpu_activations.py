"""The activations of the products and the group norm relative to their results,
down to small and far negative arguments.

u = 2^-24 is half an fp32 step.  Bounds count, relative to the result: 2^x
(ex2, 4 u), expf (2 steps, 4 u), erff (2 steps), a quotient or reciprocal (2 u),
every product and sum (1 u), and what a rounded exponent adds."""
import math

import pytest
import torch

import int8_kernel_lab_b200 as m
from operators_reference import FLOOR, HALF, U

pytestmark = pytest.mark.gpu

FORMULAS = {"silu": lambda v: v * torch.sigmoid(v),
            # Phi from erfc, which holds its digits below zero.
            "gelu": lambda v: 0.5 * v * torch.special.erfc(-v / math.sqrt(2)),
            "gelu_tanh": lambda v: v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))}


def _bound(v, activation, full):
    """Relative error in u, before the result's rounding."""
    low = (-v).clamp_min(0)
    if activation == "silu":
        # The exponent, v log2 e: the constant and the product (full: exact).
        return 8 + (0 if full else 2 * low)
    if activation == "gelu_tanh":
        # 2u = v (1.596 + 0.0714 v^2), three roundings, next to nothing above zero.
        return 8 + 1.1 + 3 * low * (1.596 + 0.0714 * low * low)
    # The fit 1.4; t 3, which reaches it up to twice; Horner's sums 4; three
    # products; the power 4; v^2 / 2 with its two roundings and the constant's half.
    tail = 1.4 + 6 + 4 + 3 + 4 + 1.25 * low * low
    if not full:
        return tail
    # Up to one: v / 2 + v^2 R, whose sum is rounded (1).  R is fitted relative to
    # the result (2.9e-8, or 0.49); its sums 2 and the two products 2.5 of v^2 R.
    # Above: what 1 - Phi is of Phi, two roundings.
    phi = 0.5 * torch.special.erfc(-v / math.sqrt(2))
    near = 1.49 + 4.5 * (v.abs() * (phi - 0.5).abs()) / (v.abs() * phi).clamp_min(1e-300)
    return torch.where(v.abs() <= 1, near, torch.where(v < 0, tail, tail * (1 - phi) / phi + 2))


def _arguments():
    """From 1e-6 to 12 on both sides, and a few that end a formula's range."""
    size = torch.logspace(-6, math.log10(12.0), 60000, dtype=torch.float64)
    ends = torch.tensor([0.0, -0.5, 0.5, 30.0, 1e4, 3e38], dtype=torch.float64)
    v = torch.cat([size, -size, torch.linspace(-6, 6, 60007, dtype=torch.float64), ends])
    return v.float().cuda()


@pytest.mark.parametrize("activation", sorted(FORMULAS))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("rows", [1, 200])   # the few-row kernel and the tiled one
def test_products_activation(cuda, rows, dtype, activation):
    v = _arguments()[::1 if rows == 1 else 20].contiguous()
    a = torch.zeros(rows, 16, dtype=torch.int8, device="cuda")
    b = torch.zeros(v.numel(), 16, dtype=torch.int8, device="cuda")
    y = m.matmul(a, b, bias=v, activation=activation, dtype=dtype)
    _check(y, v.double().expand(rows, -1), activation, dtype)


def _check(y, v, activation, dtype):
    want = FORMULAS[activation](v)
    # A reciprocal below 2^-126 is zero: the result is less than |v| times that.
    tol = U * _bound(v, activation, dtype == torch.float32) * want.abs() + v.abs() * 2.0 ** -126
    if dtype != torch.float32:
        tol = tol + (want.abs() + tol) * HALF[dtype] + FLOOR[dtype]
    far = want.abs() > torch.finfo(dtype).max          # rounds to infinity
    ok = ((y.double() - want).abs() <= tol) | (far & torch.isinf(y))
    assert bool(ok.all()), (f"{int((~ok).sum())} off, first at {float(v[~ok][0])}: "
                            f"{float(y[~ok][0])}, want {float(want[~ok][0])}")


@pytest.mark.parametrize("activation", sorted(FORMULAS))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("channels", [8192, 8190])   # in vectors, and one by one
def test_group_norms_activation(cuda, channels, dtype, activation):
    # A constant image normalises to zero: y = act(beta).
    v = _arguments()[::16][:channels].contiguous()
    x = torch.full((2, 9, channels), 2.5, device="cuda")
    y = m.group_norm(x, 2, None, v, activation=activation, dtype=dtype)
    _check(y, v.double().expand(2, 9, -1), activation, dtype)


def test_int8_results_of_the_activations(cuda):
    v = _arguments()
    v = v[v.abs() < 6]
    zero = torch.zeros(1, 16, dtype=torch.int8, device="cuda")
    step = 6 / 127
    for activation, f in FORMULAS.items():
        y = m.matmul(zero, zero.expand(v.numel(), 16).contiguous(), bias=v, activation=activation,
                     dtype=torch.int8, out_scale=step)
        want = f(v.double()) / step
        # The activation, the rounded 1 / step and the product with it.
        off = (y.double()[0] - want).abs() - 0.5
        assert bool((off <= U * (_bound(v.double(), activation, False) + 3) * want.abs() + 1e-30).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.int8], ids=str)
@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("activation", sorted(FORMULAS))
def test_ends_of_the_range(cuda, activation, rows, dtype):
    inf, most = float("inf"), torch.finfo(torch.float32).max
    v = torch.tensor([float("nan"), inf, -inf, most, -most, 2.5e38, -2.5e38, 0.0, -1e5, 1e-45] + [1.0] * 6,
                     device="cuda")
    a = torch.zeros(rows, 16, dtype=torch.int8, device="cuda")
    b = torch.zeros(16, 16, dtype=torch.int8, device="cuda")
    y = m.matmul(a, b, bias=v, activation=activation, dtype=dtype,
                 out_scale=0.5 if dtype == torch.int8 else None)
    for row in (y[0], y[-1]):
        if dtype == torch.int8:
            assert row[:9].tolist() == [0, 127, 0, 127, 0, 127, 0, 0, 0]
            continue
        assert torch.isnan(row[[0, 2]]).all() and row[1] == inf
        large = row[[3, 5]].double()
        if dtype == torch.float16:
            assert (large == inf).all()
        else:
            want = v[[3, 5]].double()
            assert ((large - want).abs() <= want * 2 * HALF[dtype]).logical_or(large == inf).all()
        assert (row[[4, 6, 7, 8]] == 0).all() and 0 <= float(row[9]) <= 1e-44
