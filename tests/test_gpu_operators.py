"""The products, the row quantisation and the group norm against their plain
64-bit forms (operators_reference.py), at the sizes, layouts and values where
they can go wrong."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import int8_kernel_lab_b200 as m
import operators_reference as ref
from int8_kernel_lab_b200 import _abi, operators

pytestmark = pytest.mark.gpu

FLOATS = [torch.bfloat16, torch.float16, torch.float32]
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(g, rows, k, extra=0):
    """int8 rows over the whole range, `extra` more bytes of pitch (garbage)."""
    pitch = (k + 15) // 16 * 16 + extra
    return torch.randint(-128, 128, (rows, pitch), generator=g, device="cuda",
                         dtype=torch.int8)[:, :k]


def _scales(g, n, about):
    return (torch.rand(n, generator=g, device="cuda") + 0.5) * about


def _operands(mm, n, k, seed, extra=0):
    g = _gen(seed)
    about = 1 / (74 * k ** 0.5)
    return dict(a=_ints(g, mm, k, extra), b=_ints(g, n, k, 2 * extra),
                row=_scales(g, mm, 1 / 74), col=_scales(g, n, about * 2),
                bias=torch.randn(n, generator=g, device="cuda"),
                residual=torch.randn(mm, n, generator=g, device="cuda"))


def _framed(mm, n, dtype, pitch_extra=0, lead=0):
    """An output view inside a larger buffer, and a check that nothing around it
    was written."""
    pitch = n + pitch_extra
    fill = 77
    buf = torch.full((lead + (mm + 2) * pitch,), fill, dtype=dtype, device="cuda")
    y = buf[lead + pitch:].as_strided((mm, n), (pitch, 1))

    def untouched():
        mask = torch.ones_like(buf, dtype=torch.bool)
        mask[lead + pitch:].as_strided((mm, n), (pitch, 1)).fill_(False)
        return bool((buf[mask] == fill).all())

    return y, untouched


@pytest.fixture(params=["auto", "single", "pair"])
def pairing(request):
    m.set_cta_pairing(request.param)
    yield request.param
    m.set_cta_pairing("auto")


SHAPES = [(1, 1, 1), (1, 4096, 512), (2, 33, 16), (3, 5, 7), (8, 1000, 2050), (16, 64, 4096),
          (17, 96, 100), (65, 31, 129), (128, 256, 128), (129, 257, 131), (200, 1000, 1040),
          (513, 640, 96), (1100, 2100, 260), (1, 500, 4100), (100, 300, 5000),
          (3, 70, 16400), (128, 512, 1536), (140, 200, 3000)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_matmul_shapes(cuda, pairing, shape):
    mm, n, k = shape
    o = _operands(mm, n, k, 1)
    for dtype in FLOATS:
        y, untouched = _framed(mm, n, dtype)
        res = o["residual"].to(dtype)
        m.launch_matmul(o["a"], o["b"], y, row_scale=o["row"], col_scale=o["col"], bias=o["bias"],
                        activation="silu", residual=res)
        assert m.device_status() == _abi.OK
        want, err = ref.product(o["a"], o["b"], o["row"], o["col"], o["bias"], "silu", res)
        ref.check(y, want, err, f"{shape} {dtype} {pairing}")
        assert untouched()


@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("dtype", FLOATS + [torch.int8], ids=str)
def test_matmul_epilogues(cuda, activation, dtype):
    mm, n, k = 150, 200, 144
    o = _operands(mm, n, k, 2)
    for row, col, bias in ((1, 1, 1), (0, 1, 0), (1, 0, 0), (0, 0, 1)):
        kw = dict(row_scale=o["row"] if row else None, col_scale=o["col"] if col else None,
                  bias=o["bias"] if bias else None, activation=activation)
        step = 0.02 if row and col else 40.0
        got = m.matmul(o["a"], o["b"], dtype=dtype,
                       out_scale=step if dtype == torch.int8 else None, **kw)
        want, err = ref.product(o["a"], o["b"], kw["row_scale"], kw["col_scale"], kw["bias"],
                                activation)
        if dtype == torch.int8:
            # The factor 1 / step is rounded once, the product once more.
            ref.check_int8(got, want / step, err / step + 3 * ref.U * (want / step).abs(), activation)
        elif dtype == torch.float16 and not (row and col):
            continue  # beyond fp16's range
        else:
            ref.check(got, want, err, activation)


@pytest.mark.parametrize("dtype", FLOATS + [torch.int8], ids=str)
@pytest.mark.parametrize("layout", [(0, 0), (1, 0), (0, 1), (13, 3), (16, 0)], ids=str)
def test_matmul_pitches_and_offsets(cuda, layout, dtype):
    extra, lead = layout
    mm, n, k = 70, 83, 200
    o = _operands(mm, n, k, 3, extra=32)
    y, untouched = _framed(mm, n, dtype, extra, lead)
    res = None
    if dtype != torch.int8:
        res, _ = _framed(mm, n, dtype, extra + 5, lead)
        res.copy_(o["residual"])
    step = 0.03 if dtype == torch.int8 else None
    m.launch_matmul(o["a"], o["b"], y, row_scale=o["row"], col_scale=o["col"], residual=res,
                    out_scale=step)
    want, err = ref.product(o["a"], o["b"], o["row"], o["col"], residual=res)
    if dtype == torch.int8:
        ref.check_int8(y, want / step, err / step + 3 * ref.U * (want / step).abs())
    else:
        ref.check(y, want, err)
    assert untouched() and m.device_status() == _abi.OK


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
def test_matmul_residual_in_place(cuda, pairing, dtype):
    o = _operands(300, 520, 64, 4)
    y = o["residual"].to(dtype)
    before = y.clone()
    m.launch_matmul(o["a"], o["b"], y, row_scale=o["row"], col_scale=o["col"], residual=y)
    want, err = ref.product(o["a"], o["b"], o["row"], o["col"], residual=before)
    ref.check(y, want, err)


def test_matmul_longest_sum_is_exact(cuda):
    k = 131071
    a = torch.full((2, 131072), -128, dtype=torch.int8, device="cuda")[:, :k]
    b = torch.full((3, 131072), -128, dtype=torch.int8, device="cuda")[:, :k]
    b[1].fill_(127)
    y = m.matmul(a, b, dtype=torch.float32)
    want, err = ref.product(a, b)
    assert want[0, 0] == 131071 * 16384
    ref.check(y, want, err)


def test_matmul_nan_and_infinite_scales_stay_in_their_rows(cuda):
    o = _operands(40, 50, 64, 5)
    row = o["row"].clone()
    row[3], row[7] = float("nan"), float("inf")
    y = m.matmul(o["a"], o["b"], row_scale=row, col_scale=o["col"], dtype=torch.float32)
    assert bool(torch.isnan(y[3]).all()) and not bool(torch.isfinite(y[7]).any())
    keep = [i for i in range(40) if i not in (3, 7)]
    want, err = ref.product(o["a"][keep], o["b"], row[keep], o["col"])
    ref.check(y[keep], want, err)
    q = m.matmul(o["a"], o["b"], row_scale=row, col_scale=o["col"], dtype=torch.int8, out_scale=0.1)
    assert bool((q[3] == 0).all())


def test_matmul_of_nothing(cuda):
    a = torch.empty(0, 64, dtype=torch.int8, device="cuda")
    b = torch.zeros(8, 64, dtype=torch.int8, device="cuda")
    assert m.matmul(a, b).shape == (0, 8)
    assert m.matmul(b, a).shape == (8, 0)
    before = m.launch_count()
    assert m.quantize_rows(torch.empty(0, 64, device="cuda"))[0].shape == (0, 64)
    assert m.group_norm(torch.empty(2, 0, 32, device="cuda"), 4).shape == (2, 0, 32)
    assert m.launch_count() == before


def _grouped_case(sizes, n, k, seed, first=0, behind=0):
    g = _gen(seed)
    e, total = len(sizes), first + sum(sizes) + behind
    b = _ints(g, e * n, k)
    b = b.as_strided((e, n, k), (n * b.stride(0), b.stride(0), 1))
    offsets = torch.tensor([first + sum(sizes[:i]) for i in range(e + 1)], dtype=torch.int32,
                           device="cuda")
    return dict(a=_ints(g, total, k), b=b, offsets=offsets, row=_scales(g, total, 1 / 74),
                col=_scales(g, e * n, 2 / (74 * k ** 0.5)).view(e, n),
                bias=torch.randn(e, n, generator=g, device="cuda"))


def _check_grouped(o, y, before, bounds, dtype, step=None):
    for e, (lo, hi) in enumerate(bounds):
        want, err = ref.product(o["a"][lo:hi], o["b"][e], o["row"][lo:hi], o["col"][e],
                                o["bias"][e], "silu")
        if dtype == torch.int8:
            ref.check_int8(y[lo:hi], want / step, err / step + 3 * ref.U * (want / step).abs())
        else:
            ref.check(y[lo:hi], want, err, f"expert {e}")
    outside = torch.ones(y.shape[0], dtype=torch.bool, device="cuda")
    for lo, hi in bounds:
        outside[lo:hi] = False
    assert torch.equal(y[outside], before[outside])


@pytest.mark.parametrize("dtype", FLOATS + [torch.int8], ids=str)
@pytest.mark.parametrize("sizes,n,k,first,behind", [
    ([1], 64, 64, 0, 0),
    ([5, 0, 3, 0, 0, 1], 100, 80, 0, 0),
    ([0, 0, 200, 129, 0, 7], 257, 300, 3, 9),
    ([300, 31, 32, 33, 512], 520, 128, 0, 1),
    ([0, 0, 0], 40, 48, 2, 5),
    ([1, 0] * 60, 33, 16, 0, 0),
], ids=str)
def test_grouped_matmul(cuda, pairing, sizes, n, k, first, behind, dtype):
    o = _grouped_case(sizes, n, k, 6, first, behind)
    y, untouched = _framed(o["a"].shape[0], n, dtype)
    y.fill_(5)
    before = y.clone()
    step = 0.03 if dtype == torch.int8 else None
    m.launch_grouped_matmul(o["a"], o["b"], o["offsets"], y, row_scale=o["row"],
                            col_scale=o["col"], bias=o["bias"], activation="silu", out_scale=step)
    assert m.device_status() == _abi.OK
    ends = o["offsets"].tolist()
    _check_grouped(o, y, before, list(zip(ends, ends[1:])), dtype, step)
    assert untouched()


def test_grouped_matmul_most_experts(cuda):
    sizes = [(i * 7) % 4 for i in range(1024)]
    o = _grouped_case(sizes, 32, 32, 7)
    y = m.grouped_matmul(o["a"], o["b"], o["offsets"], row_scale=o["row"], col_scale=o["col"],
                         bias=o["bias"], activation="silu", dtype=torch.float32)
    ends = o["offsets"].tolist()
    _check_grouped(o, y, y, list(zip(ends, ends[1:])), torch.float32)


def test_grouped_matmul_reads_bad_offsets_within_bounds(cuda):
    # Each offset counts as at least its predecessor and at most the rows.
    o = _grouped_case([40, 40, 40, 40], 96, 64, 8)
    o["offsets"] = torch.tensor([-5, 50, 20, 999, 130], dtype=torch.int32, device="cuda")
    y = torch.full((160, 96), 3.0, device="cuda")
    m.launch_grouped_matmul(o["a"], o["b"], o["offsets"], y, row_scale=o["row"],
                            col_scale=o["col"], bias=o["bias"], activation="silu")
    _check_grouped(o, y, y, [(0, 50), (50, 50), (50, 160), (160, 160)], torch.float32)


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("k", [1, 7, 8, 100, 1024, 1025, 4096, 5000, 20000])
def test_quantize_rows(cuda, dtype, k):
    g = _gen(9)
    x = (torch.randn(37, k, generator=g, device="cuda") * 3).to(dtype)
    x[5] = 0
    x[6, 0] = float("inf")
    x[7, k // 2] = float("nan")
    x[8] *= 1e-3
    q, scale = m.quantize_rows(x)
    want, wscale = ref.quantized(x)
    assert torch.equal(scale.cpu().nan_to_num(-1), wscale.nan_to_num(-1))
    assert torch.equal(q.cpu(), want)
    assert q.stride(0) % 16 == 0 and float(scale[5]) == 0 and bool(torch.isnan(scale[6:8]).all())


def test_quantize_rows_of_tiny_values(cuda):
    # fp32 denormals: the scale has few bits, or none.
    x = torch.tensor([[1e-45, 0.0], [190 * 1.4e-45, -190 * 1.4e-45], [1e-38, 5e-39]], device="cuda")
    q, scale = m.quantize_rows(x)
    want, wscale = ref.quantized(x)
    assert torch.equal(scale.cpu(), wscale) and torch.equal(q.cpu(), want)


def test_quantize_rows_gathers(cuda):
    g = _gen(10)
    x = torch.randn(20, 300, generator=g, device="cuda").to(torch.bfloat16)
    index = torch.tensor([3, 3, 0, 19, -1, 20, 2**31 - 1, 7], dtype=torch.int32, device="cuda")
    q, scale = m.quantize_rows(x, index)
    want, wscale = ref.quantized(x)
    for i, r in enumerate(index.tolist()):
        if 0 <= r < 20:
            assert torch.equal(q[i].cpu(), want[r]) and float(scale[i]) == float(wscale[r])
        else:
            assert not bool(q[i].any()) and float(scale[i]) == 0


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("lead,pitch", [(0, 104), (1, 105), (3, 200)])
def test_quantize_rows_strides(cuda, dtype, lead, pitch):
    g = _gen(11)
    buf = torch.randn(lead + 30 * pitch, generator=g, device="cuda").to(dtype)
    x = buf[lead:].as_strided((30, 101), (pitch, 1))
    q = torch.full((30, 131), 99, dtype=torch.int8, device="cuda")
    scale = torch.empty(30, device="cuda")
    m.launch_quantize_rows(x, q[:, :101], scale)
    want, wscale = ref.quantized(x)
    assert torch.equal(q[:, :101].cpu(), want) and torch.equal(scale.cpu(), wscale)
    assert bool((q[:, 101:] == 99).all())


def _norm_input(g, n, p, c, dtype, mean=0.5, spread=1.0):
    x = torch.randn(n, p, c, generator=g, device="cuda") * spread + mean
    if dtype == torch.int32:
        return (x * 2000).round().to(torch.int32), _scales(g, c, 1 / 2000)
    return x.to(dtype), None


@pytest.mark.parametrize("source", FLOATS + [torch.int32], ids=str)
@pytest.mark.parametrize("n,p,c,groups", [(1, 1, 2, 1), (2, 1, 64, 32), (1, 196, 256, 32),
                                          (3, 77, 320, 32), (2, 50, 30, 5), (5, 9, 7, 7),
                                          (1, 1000, 33, 1), (2, 64, 2560, 32), (1, 3, 8192, 8),
                                          (70, 20, 48, 3), (1, 40, 4096, 4096),
                                          (2, 5, 8192, 4096), (150, 30, 72, 9)])
def test_group_norm(cuda, source, n, p, c, groups):
    g = _gen(12)
    x, scale = _norm_input(g, n, p, c, source)
    gamma, beta = _scales(g, c, 1.0), torch.randn(c, generator=g, device="cuda")
    want, err = ref.norm(x, groups, gamma, beta, 1e-5, "silu", scale)
    for dtype in FLOATS:
        y = m.group_norm(x, groups, gamma, beta, activation="silu", scale=scale, dtype=dtype)
        ref.check(y, want, err, str(dtype))
    step = 0.04
    y = m.group_norm(x, groups, gamma, beta, activation="silu", scale=scale, dtype=torch.int8,
                     out_scale=step)
    ref.check_int8(y, want / step, err / step + 3 * ref.U * (want / step).abs())


@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("gamma,beta", [(0, 0), (1, 0), (0, 1)])
def test_group_norm_epilogues(cuda, activation, gamma, beta):
    g = _gen(13)
    x, _ = _norm_input(g, 2, 40, 64, torch.float32)
    gamma = _scales(g, 64, 2.0) if gamma else None
    beta = torch.randn(64, generator=g, device="cuda") if beta else None
    y = m.group_norm(x, 8, gamma, beta, eps=1e-3, activation=activation)
    want, err = ref.norm(x, 8, gamma, beta, 1e-3, activation)
    ref.check(y, want, err)


def test_group_norm_far_mean(cuda):
    # A mean a thousand deviations away leaves ten bits of the input's 24.
    g = _gen(14)
    x, _ = _norm_input(g, 2, 500, 64, torch.float32, mean=1000.0)
    want, err = ref.norm(x, 4)
    ref.check(m.group_norm(x, 4), want, err)


def test_group_norm_constant_and_not_finite_groups(cuda):
    x = torch.randn(2, 30, 32, generator=_gen(15), device="cuda")
    x[0, :, 0:8] = 3.25
    x[1, 4, 9] = float("nan")
    x[1, 5, 17] = float("inf")
    y = m.group_norm(x, 4)
    assert bool((y[0, :, 0:8] == 0).all())
    assert bool(torch.isnan(y[1, :, 8:24]).all())
    rest = y.clone()
    rest[1, :, 8:24] = 0
    assert bool(torch.isfinite(rest).all())
    x = torch.nan_to_num(x, nan=0.0, posinf=0.0)
    want, err = ref.norm(x, 4)
    ref.check(y[0], want[0], err[0])
    ref.check(y[1, :, 24:], want[1, :, 24:], err[1, :, 24:])


@pytest.mark.parametrize("c,pitch,lead", [(32, 48, 0), (32, 33, 0), (24, 40, 3), (21, 30, 1)])
@pytest.mark.parametrize("dtype", FLOATS + [torch.int8], ids=str)
def test_group_norm_strides(cuda, c, pitch, lead, dtype):
    # A slice of the channels of a wider tensor, and into one.
    g = _gen(16)
    n, h, w = 2, 5, 6
    wide = torch.randn(lead + n * h * w * pitch, generator=g, device="cuda")
    x = wide[lead:].as_strided((n, h, w, c), (h * w * pitch, w * pitch, pitch, 1))
    out = torch.full((lead + n * h * w * pitch,), 77, dtype=dtype, device="cuda")
    y = out[lead:].as_strided(x.shape, x.stride())
    step = 0.05 if dtype == torch.int8 else None
    ws = torch.empty(m.group_norm_workspace_bytes(x, 3 if c % 3 == 0 else 4, y), dtype=torch.uint8,
                     device="cuda")
    groups = 3 if c % 3 == 0 else 4
    m.launch_group_norm(x, groups, y, workspace=ws, workspace_bytes=ws.numel(), out_scale=step)
    want, err = ref.norm(x.reshape(n, h * w, c), groups)
    got = y.reshape(n, h * w, c)
    if step:
        ref.check_int8(got, want / step, err / step + 3 * ref.U * (want / step).abs())
    else:
        ref.check(got, want, err)
    y.fill_(77)
    assert bool((out == 77).all())


def test_group_norm_in_place_and_deterministic(cuda):
    g = _gen(17)
    x, _ = _norm_input(g, 4, 900, 96, torch.bfloat16)
    want = m.group_norm(x, 8, activation="gelu")
    for _ in range(3):
        y = x.clone()
        ws = torch.empty(m.group_norm_workspace_bytes(y, 8, y), dtype=torch.uint8, device="cuda")
        m.launch_group_norm(y, 8, y, activation="gelu", workspace=ws, workspace_bytes=ws.numel())
        assert torch.equal(y, want)


def test_group_norm_channel_worth_nothing(cuda):
    # A channel whose step is worth 0 is zero throughout, and still has a place
    # in its group's statistics.
    g = _gen(34)
    x, scale = _norm_input(g, 2, 90, 40, torch.int32)
    scale[[0, 13]] = 0
    beta = torch.randn(40, generator=g, device="cuda")
    y = m.group_norm(x, 5, beta=beta, scale=scale, activation="silu", dtype=torch.float32)
    want, err = ref.norm(x, 5, None, beta, 1e-5, "silu", scale)
    ref.check(y, want, err)


def test_elements_past_two_to_the_31(cuda):
    # Rows, pitches and results whose element offsets do not fit 32 bits.
    g = _gen(35)
    rows, n = 40000, 60000                       # 2.4e9 results
    o = _operands(rows, n, 16, 36)
    y = m.matmul(o["a"], o["b"], row_scale=o["row"], col_scale=o["col"], bias=o["bias"])
    at = torch.tensor([0, 1, 35790, 35791, 35792, rows - 1], device="cuda")
    want, err = ref.product(o["a"][at], o["b"], o["row"][at], o["col"], o["bias"])
    ref.check(y[at], want, err)
    q, scale = m.quantize_rows(y)
    wq, wscale = ref.quantized(y[at])
    assert torch.equal(q[at].cpu(), wq) and torch.equal(scale[at].cpu(), wscale)
    back = m.matmul(q, q[:5], row_scale=scale, dtype=torch.float32)   # reads 2.4e9 bytes of a
    want, err = ref.product(q[at], q[:5], scale[at])
    ref.check(back[at], want, err)
    index = torch.tensor([rows - 1, 35792], dtype=torch.int32, device="cuda")
    assert torch.equal(m.quantize_rows(y, index)[0], q[index.long()])
    del q, back
    x = y.view(2, -1, 64)                        # 1.2e9 elements an image
    z = m.group_norm(x, 1, activation="relu")
    mean = x.float().mean((1, 2), keepdim=True, dtype=torch.float64)
    var = torch.stack([(i.float() - c.float()).square().mean(dtype=torch.float64)
                       for i, c in zip(x, mean)]).view(2, 1, 1)
    for sl in (slice(0, 1000), slice(-1000, None)):
        want = ((x[:, sl].double() - mean) / (var + 1e-5).sqrt()).clamp_min(0).cpu()
        # 18.7e6 pixels over 296 CTAs of 64 threads a column: runs of 1000 additions.
        ref.check(z[:, sl], want, want.abs() * 2000 * ref.U + 2000 * ref.U, "norm")


def test_operators_from_two_streams_at_once(cuda):
    args = [_block_inputs(40 + i) for i in range(2)]
    want = [_block(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_block(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
    assert m.device_status() == _abi.OK


def test_first_call_of_a_process_may_be_captured(cuda):
    code = """
import torch, int8_kernel_lab_b200 as m
a = torch.ones(40, 64, dtype=torch.int8, device="cuda")
x = torch.randn(40, 64, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    q, s = m.quantize_rows(x)
    y = m.matmul(a, a, residual=None, dtype=torch.float32)
    z = m.group_norm(x.view(2, 20, 64), 4)
g.replay()
torch.cuda.synchronize()
assert torch.equal(y, torch.full((40, 40), 64.0, device="cuda")), y
assert torch.equal(q, m.quantize_rows(x)[0]) and torch.equal(z, m.group_norm(x.view(2, 20, 64), 4))
"""
    root = Path(__file__).resolve().parent.parent
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True,
                          timeout=120)
    assert done.returncode == 0, done.stderr[-2000:]


def _block(x, w1, c1, w2, c2, gamma, beta):
    """Norm to int8, a widening and a narrowing product with the residual."""
    q = m.group_norm(x, 8, gamma, beta, activation="silu", dtype=torch.int8, out_scale=0.03)
    rows = q.view(-1, x.shape[-1])
    h = m.matmul(rows, w1, col_scale=c1 * 0.03, activation="gelu", dtype=torch.bfloat16)
    hq, row = m.quantize_rows(h)
    return m.matmul(hq, w2, row_scale=row, col_scale=c2, residual=x.view(rows.shape))


def _block_inputs(seed):
    g = _gen(seed)
    c, hidden = 96, 400
    x = torch.randn(2, 65, c, generator=g, device="cuda").to(torch.bfloat16)
    w1, c1 = m.quantize_rows(torch.randn(hidden, c, generator=g, device="cuda") / c ** 0.5)
    w2, c2 = m.quantize_rows(torch.randn(c, hidden, generator=g, device="cuda") / hidden ** 0.5)
    return x, w1, c1, w2, c2, _scales(g, c, 1.0), torch.randn(c, generator=g, device="cuda")


def test_operators_in_a_block(cuda):
    args = _block_inputs(18)
    x, w1, c1, w2, c2, gamma, beta = args
    got = _block(*args)
    # Each step against its plain form on what the step before really gave.
    q = m.group_norm(x, 8, gamma, beta, activation="silu", dtype=torch.int8, out_scale=0.03)
    z, err = ref.norm(x, 8, gamma, beta, 1e-5, "silu")
    ref.check_int8(q, z / 0.03, err / 0.03 + 3 * ref.U * (z / 0.03).abs())
    h = m.matmul(q.view(-1, 96), w1, col_scale=c1 * 0.03, activation="gelu")
    ref.check(h, *ref.product(q.view(-1, 96), w1, None, c1 * 0.03, None, "gelu"))
    hq, row = m.quantize_rows(h)
    want, wrow = ref.quantized(h)
    assert torch.equal(hq.cpu(), want) and torch.equal(row.cpu(), wrow)
    ref.check(got, *ref.product(hq, w2, row, c2, residual=x.view(-1, 96)))


def test_conv_output_through_norm_to_conv(cuda):
    # int32 output of a convolution -> norm + activation -> int8 input of the next.
    shape = m.ConvShape(2, 14, 14, 64, 96, 3, 3, 1, 1)
    g = _gen(19)
    x = torch.randint(-128, 128, (2, 14, 14, 64), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-128, 128, (96, 3, 3, 64), generator=g, device="cuda", dtype=torch.int8)
    b = torch.randint(-1000, 1000, (96,), generator=g, device="cuda", dtype=torch.int32)
    acc = m.conv2d(shape, x, w, b).view(2, 14, 14, 96)
    scale = _scales(g, 96, 1e-5)
    q = m.group_norm(acc, 8, scale=scale, activation="relu", dtype=torch.int8, out_scale=0.03)
    z, err = ref.norm(acc.view(2, 196, 96), 8, activation="relu", scale=scale)
    ref.check_int8(q.view(2, 196, 96), z / 0.03, err / 0.03 + 3 * ref.U * (z / 0.03).abs())
    one = m.ConvShape(2, 14, 14, 96, 32, 1, 1)
    w1 = torch.randint(-128, 128, (32, 96), generator=g, device="cuda", dtype=torch.int8)
    zero = torch.zeros(32, dtype=torch.int32, device="cuda")
    y = m.conv2d(one, q, w1, zero).view(-1, 32)
    assert torch.equal(y.double(), q.view(-1, 96).double() @ w1.double().t())
    # The same 1x1 convolution as a product.
    assert torch.equal(m.matmul(q.view(-1, 96), w1, dtype=torch.float32), y.float())


def test_operators_on_another_stream_and_captured(cuda):
    args, other = _block_inputs(20), _block_inputs(21)
    want, want_other = _block(*args), _block(*other)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _block(*args)
    side.synchronize()
    assert torch.equal(got, want)
    x = args[0]
    y = m.group_norm(x, 8, stream=side)
    side.synchronize()
    assert torch.equal(y, m.group_norm(x, 8))
    graphs = []
    for a in (args, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _block(*a)
        graphs.append((graph, out))
    for _ in range(2):
        for graph, out in graphs:
            out.zero_()
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want_other)
    # New values at the same addresses.
    args[0].copy_(other[0])
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], _block(*args))
    assert m.device_status() == _abi.OK


def test_grouped_matmul_captured_reads_new_offsets(cuda):
    o = _grouped_case([30, 50, 0, 20], 64, 96, 22)
    y = torch.zeros(100, 64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.launch_grouped_matmul(o["a"], o["b"], o["offsets"], y, row_scale=o["row"],
                                col_scale=o["col"], bias=o["bias"], activation="silu")
    for ends in ([0, 30, 80, 80, 100], [0, 0, 1, 99, 100], [10, 10, 10, 10, 40]):
        o["offsets"].copy_(torch.tensor(ends, dtype=torch.int32))
        y.fill_(4.0)
        before = y.clone()
        graph.replay()
        torch.cuda.synchronize()
        _check_grouped(o, y, before, list(zip(ends, ends[1:])), torch.float32)


def test_compiled_and_checked_calls_agree(cuda, monkeypatch):
    # The calls through torch_calls and those through the Python checks launch
    # the same kernels on the same arguments, strided and odd ones too.
    def results():
        out = []
        o = _operands(33, 50, 70, 30, extra=16)
        y, _ = _framed(33, 50, torch.float16, 3, 1)
        m.launch_matmul(o["a"], o["b"], y, row_scale=o["row"], col_scale=o["col"])
        out += [y, m.matmul(o["a"][:1], o["b"], bias=o["bias"], activation="gelu"),
                m.matmul(o["a"], o["b"], col_scale=o["col"], dtype=torch.int8, out_scale=0.5),
                m.matmul(o["a"], o["b"], residual=o["residual"][:, :50], dtype=torch.float32)]
        e = _grouped_case([9, 0, 5], 40, 50, 31)
        out += [m.grouped_matmul(e["a"], e["b"], e["offsets"], row_scale=e["row"],
                                 col_scale=e["col"], bias=e["bias"], activation="relu")]
        x = torch.randn(20, 45, generator=_gen(32), device="cuda")
        index = torch.tensor([4, 4, 19, 0], dtype=torch.int32, device="cuda")
        q, scale = torch.zeros(20, 45, dtype=torch.int8, device="cuda"), torch.zeros(20, device="cuda")
        m.launch_quantize_rows(x[:, ::1], q, scale)
        out += [q, scale, *m.quantize_rows(x, index), *m.quantize_rows(x[:, 3:17])]
        z = torch.randn(2, 6, 7, 24, generator=_gen(33), device="cuda").to(torch.bfloat16)
        out += [m.group_norm(z, 4, activation="silu"), m.group_norm(z[..., 8:], 2, dtype=torch.float32),
                m.group_norm(z, 3, dtype=torch.int8, out_scale=0.1)]
        return out

    assert operators._calls is not None, "torch_calls.so was not built"
    fast = results()
    monkeypatch.setattr(operators, "_calls", None)
    slow = results()
    for a, b in zip(fast, slow):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride()
        assert torch.equal(a, b)


def test_timed_out_waits_are_reported(cuda):
    o = _operands(64, 64, 256, 23)
    m.set_wait_limit_ns(20_000_000)
    m.debug_starve_producer(True)
    try:
        m.matmul(o["a"], o["b"])
        assert m.device_status() == _abi.DEVICE_TIMEOUT
    finally:
        m.debug_starve_producer(False)
        m.set_wait_limit_ns(0)
    y = m.matmul(o["a"], o["b"], dtype=torch.float32)
    ref.check(y, *ref.product(o["a"], o["b"]))
    assert m.device_status() == _abi.OK
