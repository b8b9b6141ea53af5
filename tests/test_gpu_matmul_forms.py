"""Products whose CTAs walk several tiles, in every form: accumulators and ring
slots used again, the residual read a tile ahead, a column tile of b that stays.
Every element is compared, with a product in 64 bits on the GPU."""
import pytest
import torch

import int8_kernel_lab_b200 as m
import operators_reference as ref
from int8_kernel_lab_b200 import _abi
from test_gpu_operators import _framed, _gen, _grouped_case, _operands
from test_matmul_forms_cpu import PAIRS, PLAIN, RESIDENT, form, tiles_per_cta

pytestmark = pytest.mark.gpu
SIZES = [s[:3] for s in [*RESIDENT, *PLAIN, *PAIRS]] + [(7000, 2100, 70)]


def _product(a, b, row, col, bias=None, activation="none", residual=None):
    """(value, error) as operators_reference.product has them, on the GPU."""
    p = (a.double() @ b.double().t()) * col.double() * row.double()[:, None]
    v = p if bias is None else p + bias.double()
    err = ref.act_error(v, ref.U * (2.01 * p.abs() + 1.01 * v.abs()), activation)
    y = ref.act(v, activation)
    if residual is not None:
        y = y + residual.double()
        err = err + 1.01 * ref.U * y.abs()
    return y, err


def _check(got, want, err, step=None):
    got = got.double()
    if step is not None:
        want, err = want / step, err / step + 3 * ref.U * (want / step).abs()
        ok = (got >= (want - err - 0.5).clamp(-128, 127)) & (got <= (want + err + 0.5).clamp(-128, 127))
    else:
        ok = (got - want).abs() <= err
    assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} off, first at {(~ok).nonzero()[0].tolist()}"


def _rounded(want, err, dtype):
    return err + (want.abs() + err) * ref.HALF[dtype] + ref.FLOOR[dtype]


@pytest.fixture(params=["auto", "single", "pair"])
def pairing(request):
    m.set_cta_pairing(request.param)
    yield request.param
    m.set_cta_pairing("auto")


def test_the_device_has_the_sms_that_the_sizes_are_for(cuda):
    assert torch.cuda.get_device_properties(0).multi_processor_count == 148
    assert sum(tiles_per_cta(*s) >= 2 for s in SIZES) >= 8
    assert form(20000, 320, 320, 0)["resident"]


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_every_element(cuda, pairing, size):
    mm, n, k = size
    o = _operands(mm, n, k, 80)
    args = dict(row_scale=o["row"], col_scale=o["col"])
    # fp32 with everything, rows at an odd pitch
    y, untouched = _framed(mm, n, torch.float32, 3, 1)
    res = o["residual"]
    m.launch_matmul(o["a"], o["b"], y, bias=o["bias"], activation="silu", residual=res, **args)
    want, err = _product(o["a"], o["b"], o["row"], o["col"], o["bias"], "silu", res)
    _check(y, want, _rounded(want, err, torch.float32))
    assert untouched()
    # 16 bits, the residual in place
    for dtype in (torch.bfloat16, torch.float16):
        y = res.to(dtype)
        want, err = _product(o["a"], o["b"], o["row"], o["col"], residual=y)
        m.launch_matmul(o["a"], o["b"], y, residual=y, **args)
        _check(y, want, _rounded(want, err, dtype))
    # int8
    q = m.matmul(o["a"], o["b"], bias=o["bias"], dtype=torch.int8, out_scale=0.03, **args)
    want, err = _product(o["a"], o["b"], o["row"], o["col"], o["bias"])
    _check(q, want, err, 0.03)
    assert m.device_status() == _abi.OK


@pytest.mark.parametrize("size", [(20000, 320, 320), (6000, 1500, 2100), (4100, 5000, 4100)], ids=str)
def test_again_and_captured(cuda, size):
    o = _operands(*size, 81)
    args = dict(row_scale=o["row"], col_scale=o["col"], bias=o["bias"], residual=o["residual"].bfloat16())
    want = m.matmul(o["a"], o["b"], **args)
    for _ in range(10):
        assert torch.equal(m.matmul(o["a"], o["b"], **args), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m.matmul(o["a"], o["b"], **args)
    for _ in range(2):
        y.zero_()
        graph.replay()
        assert torch.equal(y, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.int8], ids=str)
@pytest.mark.parametrize("sizes,n,k", [([3000, 0, 129, 5000, 1], 1100, 700),
                                       ([700] * 12 + [31] * 9, 2000, 900)], ids=str)
def test_grouped_in_several_waves(cuda, pairing, sizes, n, k, dtype):
    o = _grouped_case(sizes, n, k, 82, 2, 5)
    rows = o["a"].shape[0]
    y = m.grouped_matmul(o["a"], o["b"], o["offsets"], row_scale=o["row"], col_scale=o["col"],
                         bias=o["bias"], activation="relu", dtype=dtype,
                         out_scale=0.03 if dtype == torch.int8 else None)
    assert y.shape == (rows, n)
    ends = o["offsets"].tolist()
    for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
        want, err = _product(o["a"][lo:hi], o["b"][e], o["row"][lo:hi], o["col"][e], o["bias"][e], "relu")
        if dtype == torch.int8:
            _check(y[lo:hi], want, err, 0.03)
        else:
            _check(y[lo:hi], want, _rounded(want, err, dtype))
    assert m.device_status() == _abi.OK
