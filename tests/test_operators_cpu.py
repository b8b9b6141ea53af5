"""Refusals of the products, the row quantisation and the group norm: statuses
of the C entry points and errors of the Python ones, without a GPU."""
import ctypes

import pytest
import torch

import int8_kernel_lab_b200 as m
from int8_kernel_lab_b200 import _abi, operators

LIB = _abi.lib
A = 1 << 20  # an aligned address nothing dereferences
NO_GPU = (_abi.CUDA_ERROR, _abi.UNSUPPORTED_DEVICE)


def _matmul(**change):
    d = _abi.CMatmul(m=8, n=24, k=30, lda=32, ldb=32, ldy=24, ldr=24, y_dtype=_abi.BF16)
    for name, value in change.items():
        setattr(d, name, value)
    return d


def _launch(d, a=A, b=A, y=A):
    return LIB.int8conv_launch_matmul(ctypes.byref(d), a, b, y, None)


@pytest.mark.parametrize("change", [
    dict(m=-1), dict(n=-1), dict(k=0), dict(k=131072, lda=131072, ldb=131072), dict(lda=16),
    dict(lda=40), dict(ldb=31), dict(ldb=40), dict(ldy=23), dict(ldr=23, residual=A),
    dict(activation=5), dict(activation=-1), dict(y_dtype=_abi.INT32), dict(y_dtype=9),
    dict(y_dtype=_abi.INT8), dict(y_dtype=_abi.INT8, out_scale=-1.0),
    dict(y_dtype=_abi.INT8, out_scale=float("nan")), dict(y_dtype=_abi.INT8, out_scale=1e-45),
    dict(y_dtype=_abi.INT8, out_scale=1.0, residual=A), dict(m=1 << 31), dict(n=1 << 40),
    dict(lda=1 << 40),
])
def test_matmul_arguments(change):
    assert _launch(_matmul(**change)) == _abi.BAD_ARGUMENT
    d = _matmul(**change)
    assert LIB.int8conv_launch_grouped_matmul(ctypes.byref(d), A, A, 1024, A, 2, A,
                                              None) == _abi.BAD_ARGUMENT


@pytest.mark.parametrize("pointers", [dict(a=None), dict(b=None), dict(y=None), dict(a=A + 8),
                                      dict(b=A + 1), dict(y=A + 1)])
def test_matmul_pointers(pointers):
    assert _launch(_matmul(), **pointers) == _abi.BAD_POINTER


@pytest.mark.parametrize("change", [dict(row_scale=A + 2), dict(col_scale=A + 1),
                                    dict(bias=A + 3), dict(residual=A + 1)])
def test_matmul_vectors(change):
    assert _launch(_matmul(**change)) == _abi.BAD_POINTER


def test_a_null_descriptor_is_refused():
    assert LIB.int8conv_launch_matmul(None, A, A, A, None) == _abi.BAD_ARGUMENT
    assert LIB.int8conv_launch_group_norm(None, A, A, None, 0, None) == _abi.BAD_ARGUMENT
    assert LIB.int8conv_group_norm_workspace_bytes(None) == 0


def test_empty_products_need_no_device():
    assert _launch(_matmul(m=0), None, None, None) == _abi.OK
    assert _launch(_matmul(n=0, ldy=0), None, None, None) == _abi.OK


def test_well_formed_calls_reach_the_device():
    if torch.cuda.is_available():
        pytest.skip("made-up addresses")
    assert _launch(_matmul()) in NO_GPU
    d = _matmul()
    assert LIB.int8conv_launch_grouped_matmul(ctypes.byref(d), A, A, 1024, A, 2, A, None) in NO_GPU
    assert LIB.int8conv_launch_quantize_rows(4, 8, _abi.BF16, A, 4, 8, None, A, 8, A, None) in NO_GPU
    n = _norm()
    size = LIB.int8conv_group_norm_workspace_bytes(ctypes.byref(n))
    assert LIB.int8conv_launch_group_norm(ctypes.byref(n), A, A, A, size, None) in NO_GPU


@pytest.mark.parametrize("stride,groups,offsets,status", [
    (1024, 0, A, _abi.BAD_ARGUMENT), (1024, 1025, A, _abi.BAD_ARGUMENT),
    (1000, 2, A, _abi.BAD_ARGUMENT), (0, 2, A, _abi.BAD_ARGUMENT), (-1024, 2, A, _abi.BAD_ARGUMENT),
    (1024, 2, None, _abi.BAD_POINTER), (1024, 2, A + 2, _abi.BAD_POINTER)])
def test_grouped_arguments(stride, groups, offsets, status):
    d = _matmul()
    assert LIB.int8conv_launch_grouped_matmul(ctypes.byref(d), A, A, stride, offsets, groups, A,
                                              None) == status


def test_grouped_takes_no_residual():
    d = _matmul(residual=A)
    assert LIB.int8conv_launch_grouped_matmul(ctypes.byref(d), A, A, 1024, A, 2, A,
                                              None) == _abi.BAD_ARGUMENT


@pytest.mark.parametrize("args,status", [
    ((-1, 8, 0, A, 4, 8, None, A, 8, A), _abi.BAD_ARGUMENT),
    ((4, 0, 0, A, 4, 8, None, A, 8, A), _abi.BAD_ARGUMENT),
    ((4, 8, _abi.INT8, A, 4, 8, None, A, 8, A), _abi.BAD_ARGUMENT),
    ((4, 8, 0, A, 4, 7, None, A, 8, A), _abi.BAD_ARGUMENT),
    ((4, 8, 0, A, 4, 8, None, A, 7, A), _abi.BAD_ARGUMENT),
    ((4, 8, 0, A, 3, 8, None, A, 8, A), _abi.BAD_ARGUMENT),   # too few rows
    ((4, 8, 0, A, -1, 8, A, A, 8, A), _abi.BAD_ARGUMENT),
    ((4, 8, 0, None, 4, 8, None, A, 8, A), _abi.BAD_POINTER),
    ((4, 8, 0, A, 4, 8, None, None, 8, A), _abi.BAD_POINTER),
    ((4, 8, 0, A, 4, 8, None, A, 8, None), _abi.BAD_POINTER),
    ((4, 8, 0, A + 1, 4, 8, None, A, 8, A), _abi.BAD_POINTER),
    ((4, 8, 0, A, 4, 8, A + 2, A, 8, A), _abi.BAD_POINTER),
    ((0, 8, 0, None, 0, 8, None, None, 8, None), _abi.OK)])
def test_quantize_rows_arguments(args, status):
    assert LIB.int8conv_launch_quantize_rows(*args, None) == status


def _norm(**change):
    d = _abi.CGroupNorm(n=2, pixels=9, channels=32, groups=4, ldx=32, ldy=32, eps=1e-5,
                        x_dtype=_abi.INT32, y_dtype=_abi.BF16)
    for name, value in change.items():
        setattr(d, name, value)
    return d


@pytest.mark.parametrize("change", [
    dict(n=-1), dict(pixels=-1), dict(channels=0), dict(channels=8193, groups=1, ldx=8193, ldy=8193),
    dict(channels=4097, groups=4097, ldx=4097, ldy=4097), dict(groups=0), dict(groups=5), dict(ldx=31), dict(ldy=31), dict(x_dtype=_abi.INT8),
    dict(y_dtype=_abi.INT32), dict(eps=-1.0), dict(eps=float("nan")), dict(activation=7),
    dict(y_dtype=_abi.INT8), dict(y_dtype=_abi.INT8, out_scale=float("inf"))])
def test_group_norm_arguments(change):
    d = _norm(**change)
    assert LIB.int8conv_launch_group_norm(ctypes.byref(d), A, A, A, 1 << 20, None) == _abi.BAD_ARGUMENT
    assert LIB.int8conv_group_norm_workspace_bytes(ctypes.byref(d)) == 0


def test_group_norm_buffers():
    d = _norm()
    size = LIB.int8conv_group_norm_workspace_bytes(ctypes.byref(d))

    def call(x=A, y=A, ws=A, nbytes=size):
        return LIB.int8conv_launch_group_norm(ctypes.byref(d), x, y, ws, nbytes, None)

    assert call(x=None) == call(y=None) == call(x=A + 2) == call(y=A + 1) == _abi.BAD_POINTER
    if size:
        assert call(nbytes=size - 1) == _abi.WORKSPACE_TOO_SMALL
        assert call(ws=None) == call(ws=A + 8) == _abi.BAD_POINTER
    for empty in (dict(n=0), dict(pixels=0)):
        e = _norm(**empty)
        assert LIB.int8conv_launch_group_norm(ctypes.byref(e), None, None, None, 0, None) == _abi.OK


def test_packed_descriptors_are_the_structures():
    assert operators._MATMUL.size == ctypes.sizeof(_abi.CMatmul)
    assert operators._NORM.size == ctypes.sizeof(_abi.CGroupNorm)
    d = _abi.CMatmul.from_buffer_copy(operators._MATMUL.pack(*range(1, 14), 0.5))
    assert [getattr(d, f) for f, _ in d._fields_] == [*range(1, 14), 0.5]
    d = _abi.CGroupNorm.from_buffer_copy(
        operators._NORM.pack(1, 2, 3, 4, 5, 6, 7, 8, 9, 0.25, 10, 11, 12, 0.5))
    assert [getattr(d, f) for f, _ in d._fields_] == [1, 2, 3, 4, 5, 6, 7, 8, 9, 0.25, 10, 11, 12, 0.5]


def test_compiled_calls_decline_what_is_not_a_cuda_tensor():
    operators._load_torch()
    if operators._calls is None:
        pytest.skip("torch_calls.so was not built")
    t = torch.zeros(4, 32, dtype=torch.int8)
    none = [None] * 6
    for a in (t, 3, None, "a"):
        assert operators._calls.matmul(a, t, *none, 0, 0, None) is None
        assert operators._calls.quantize_rows(a, None, None, None) is None
        assert operators._calls.group_norm(a, 4, None, None, None, 1e-5, 0, 0, None) is None
    assert operators._calls.matmul() is None and operators._calls.group_norm(t) is None


class _Fake:
    """A CUDA tensor's outside, without a GPU."""

    def __init__(self, dtype, shape, strides=None, index=0, cuda=True):
        self.dtype, self.shape, self.is_cuda = dtype, torch.Size(shape), cuda
        strides = strides or [1]
        if len(strides) != len(shape):
            strides = [1]
            for size in reversed(shape[1:]):
                strides.insert(0, strides[0] * size)
        self._strides = tuple(strides)
        self.device = torch.device("cuda", index) if cuda else torch.device("cpu")

    def stride(self, i=None):
        return self._strides if i is None else self._strides[i]

    def numel(self):
        return self.shape.numel()

    def is_contiguous(self):
        return True

    def get_device(self):
        return self.device.index if self.is_cuda else -1

    def data_ptr(self):
        return A


@pytest.fixture
def device0(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(operators, "_stream_handle", lambda stream, device: 0)


I8, BF, F32, I32 = torch.int8, torch.bfloat16, torch.float32, torch.int32


def _mats(**change):
    t = dict(a=_Fake(I8, (4, 32)), b=_Fake(I8, (6, 32)), y=_Fake(BF, (4, 6)))
    t.update(change)
    return t


@pytest.mark.parametrize("change,message", [
    (dict(a=_Fake(BF, (4, 32))), "int8 matrix"),
    (dict(a=_Fake(I8, (4, 33))), "multiple of 16"),
    (dict(a=_Fake(I8, (4, 48))), "columns"),
    (dict(a=_Fake(I8, (4, 32), (1, 4))), "adjacent"),
    (dict(a=_Fake(I8, (4, 32), (16, 1))), "overlap"),
    (dict(b=_Fake(I8, (6, 32), index=1)), "current CUDA device"),
    (dict(a=_Fake(I8, (4, 32), cuda=False)), "CUDA tensor"),
    (dict(y=_Fake(BF, (4, 7))), "4 x 6"),
    (dict(y=_Fake(torch.float64, (4, 6))), "unsupported"),
    (dict(y=_Fake(I8, (4, 6))), "out_scale"),
    (dict(out_scale=1.0), "out_scale"),
    (dict(row_scale=_Fake(F32, (5,))), "row_scale"),
    (dict(col_scale=_Fake(BF, (6,))), "col_scale"),
    (dict(bias=_Fake(F32, (6,), index=1)), "bias"),
    (dict(residual=_Fake(F32, (4, 6))), "residual"),
    (dict(residual=_Fake(BF, (4, 5))), "residual"),
    (dict(activation="tanh"), "activation")])
def test_matmul_tensors(device0, change, message):
    t = _mats(**change)
    with pytest.raises(ValueError, match=message):
        m.launch_matmul(t.pop("a"), t.pop("b"), t.pop("y"), **t)


@pytest.mark.parametrize("change,message", [
    (dict(b=_Fake(I8, (6, 32))), "experts"),
    (dict(b=_Fake(I8, (3, 6, 32), (96, 32, 1))), "overlap"),
    (dict(offsets=_Fake(I32, (3,))), "offsets"),
    (dict(offsets=_Fake(torch.int64, (4,))), "offsets"),
    (dict(offsets=None), "offsets"),
    (dict(b=_Fake(I8, (1025, 6, 32))), "1024"),
    (dict(bias=_Fake(F32, (6,))), "bias")])
def test_grouped_tensors(device0, change, message):
    t = _mats(b=_Fake(I8, (3, 6, 32)), offsets=_Fake(I32, (4,)))
    t.update(change)
    with pytest.raises(ValueError, match=message):
        m.launch_grouped_matmul(t.pop("a"), t.pop("b"), t.pop("offsets"), t.pop("y"), **t)


@pytest.mark.parametrize("change,message", [
    (dict(x=_Fake(I32, (4, 8))), "quantize_rows"),
    (dict(x=_Fake(BF, (4, 9))), "columns"),
    (dict(x=_Fake(BF, (5, 8))), "rows"),
    (dict(q=_Fake(BF, (4, 8))), "int8"),
    (dict(scale=_Fake(F32, (5,))), "scale"),
    (dict(index=_Fake(torch.int64, (4,))), "index"),
    (dict(index=_Fake(I32, (5,))), "index")])
def test_quantize_tensors(device0, change, message):
    t = dict(x=_Fake(BF, (4, 8)), q=_Fake(I8, (4, 8)), scale=_Fake(F32, (4,)), index=None)
    t.update(change)
    with pytest.raises((ValueError, m.Int8ConvError), match=message):
        m.launch_quantize_rows(t["x"], t["q"], t["scale"], t["index"])


@pytest.mark.parametrize("change,message", [
    (dict(x=_Fake(F32, (2, 9, 32), (300, 32, 1))), "evenly"),
    (dict(x=_Fake(F32, (2, 9, 32), (288, 1, 9))), "channels-last"),
    (dict(y=_Fake(F32, (2, 9, 16))), "shape"),
    (dict(y=_Fake(I8, (2, 9, 32))), "out_scale"),
    (dict(gamma=_Fake(F32, (31,))), "gamma"),
    (dict(beta=_Fake(BF, (32,))), "beta"),
    (dict(scale=_Fake(F32, (32,), index=1)), "scale"),
    (dict(groups=5), "group_norm"),
    (dict(activation="swish"), "activation")])
def test_group_norm_tensors(device0, change, message):
    t = dict(x=_Fake(F32, (2, 9, 32)), groups=4, y=_Fake(F32, (2, 9, 32)))
    t.update(change)
    with pytest.raises((ValueError, m.Int8ConvError), match=message):
        m.launch_group_norm(t.pop("x"), t.pop("groups"), t.pop("y"), t.pop("gamma", None),
                            t.pop("beta", None), **t)
