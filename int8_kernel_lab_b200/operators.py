"""Products, row quantisation and group norm on CUDA tensors: what an int8
model runs between its convolutions (no reference counterpart).

    q, row = quantize_rows(x)                    # [m, k] floats -> int8, a scale per row
    y = matmul(q, w, row_scale=row, col_scale=col, bias=b, activation="silu", residual=r)
    y = grouped_matmul(q, experts, offsets, row_scale=row, col_scale=cols)
    z = group_norm(acc, 32, gamma, beta, scale=s, activation="silu", dtype=torch.int8, out_scale=t)

`launch_*` write into the caller's buffers and never allocate; the plain names
allocate the result (and the group norm's workspace) on the launch's stream.
Everything is asynchronous on `stream` (default: the current one), runs on the
current CUDA device and may be captured into a graph.  Results carry no
gradients.  Wrong arguments raise ValueError (types, sizes, devices) or
Int8ConvError (the library's own checks).

int8 matrices are rows of k bytes whose pitch is a multiple of 16 (the copies
into shared memory move 16-byte units): the int8 results here come that way, as
views of wider rows where k is not a multiple of 16.  A weight matrix [n, k] in
floats becomes such a matrix, with a scale per output channel, through
quantize_rows too.
"""
from __future__ import annotations

import struct

from . import _abi

# One short call to the GPU takes a few microseconds.  The calls that allocate
# their result and run on the current stream therefore go through torch_calls
# (csrc/torch_calls.cpp, where it was built for this torch and Python), which
# checks and launches a well-formed call in about one microsecond beside the
# launch itself and declines every other; what it declines, and every other
# call, takes the checks below, which name what is wrong.  They too are written
# to cost little: attributes are read once, descriptors are packed in one step,
# and torch is looked up once.
_MATMUL = struct.Struct("7q4P2if4x")        # int8conv_matmul
_NORM = struct.Struct("2q2i2q3Pf3if4x")     # int8conv_group_norm
_CALLS_PATH = _abi.LIB_PATH.parent / "torch_calls.so"
_torch = None
_DTYPES: dict = {}
_raw_stream = None
_calls = None


def _load_calls(torch):
    """The compiled calls; None where they were not built, and, with a warning,
    where they were built for another torch or Python: they read its tensors as
    they lie in memory.  The checks in Python need no such match."""
    if not _CALLS_PATH.exists():
        return None
    import importlib.util
    import sys
    import warnings

    here = f"torch {torch.__version__}, Python {sys.version_info[0]}.{sys.version_info[1]}"
    try:
        spec = importlib.util.spec_from_file_location("torch_calls", _CALLS_PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        wrong = "" if module.built_for == here else f"was built for {module.built_for}"
    except (ImportError, OSError, AttributeError) as e:
        wrong = f"does not load ({e})"
    if wrong:
        warnings.warn(f"{_CALLS_PATH} {wrong}, this is {here}: the operators' calls take longer "
                      "until it is built again", RuntimeWarning, stacklevel=2)
        return None
    module.on_failure(_abi.check)
    return module


def _load_torch():
    global _torch, _raw_stream, _calls
    import torch

    _calls = _load_calls(torch)
    _DTYPES.update({getattr(torch, name): code for name, code in _abi.DTYPES.items()})
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    _torch = torch
    return torch


def _device_index() -> int:
    return (_torch or _load_torch()).cuda.current_device()


def _stream_handle(stream, device: int) -> int:
    if stream is None:
        if _raw_stream is not None:
            return _raw_stream(device)
        return _torch.cuda.current_stream(device).cuda_stream
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _fail(name: str, want: str, t) -> None:
    if t is None:
        raise ValueError(f"{name}: expected {want}, got None")
    raise ValueError(f"{name}: expected {want}, got {t.dtype} {tuple(t.shape)} with strides "
                     f"{tuple(t.stride())} on {t.device}")


def _dtype_code(dtype) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"unsupported type {dtype}")
    return code


def _pack(descriptor: struct.Struct, *fields) -> bytes:
    try:
        return descriptor.pack(*fields)
    except struct.error as e:
        raise ValueError(f"an argument is out of range: {e}") from None


def _activation(name: str) -> int:
    code = _abi.ACTIVATIONS.get(name)
    if code is None:
        raise ValueError(f"activation: expected one of {sorted(_abi.ACTIVATIONS)}, got {name!r}")
    return code


def _misplaced(name: str, t, device: int) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor, got one on {t.device}")
    raise ValueError(f"{name} on {t.device}, but the current CUDA device is cuda:{device}: "
                     f"launch under torch.cuda.device({t.device.index}) or move the buffers")


def _vector(name: str, t, count: int, device: int, dtype=None) -> int:
    """Address of an optional contiguous vector of `count` entries (fp32)."""
    if t is None:
        return 0
    if dtype is None:
        dtype = _torch.float32
    if t.dtype != dtype or t.numel() != count or not t.is_contiguous():
        _fail(name, f"a contiguous {dtype} tensor of {count} elements", t)
    if t.get_device() != device:
        _misplaced(name, t, device)
    return t.data_ptr()


def _matrix(name: str, t, device: int):
    """(address, rows, columns, pitch) of a matrix with adjacent columns."""
    shape = t.shape
    if len(shape) != 2:
        _fail(name, "a matrix", t)
    rows, cols = shape
    pitch, unit = t.stride()
    if unit != 1 and cols > 1:
        _fail(name, "a matrix whose columns are adjacent", t)
    if t.get_device() != device:
        _misplaced(name, t, device)
    if rows <= 1:
        pitch = cols     # one row has no pitch of its own
    elif pitch < cols:
        _fail(name, "rows that do not overlap", t)
    return t.data_ptr(), rows, cols, pitch


def _int8_matrix(name: str, t, device: int):
    if t.dtype != _torch.int8:
        _fail(name, "an int8 matrix", t)
    ptr, rows, cols, pitch = _matrix(name, t, device)
    if pitch & 15:
        if rows > 1:
            raise ValueError(f"{name}: rows are {pitch} bytes apart, which is not a multiple of 16 "
                             "(quantize_rows returns rows that are)")
        pitch = (pitch + 15) & -16
    return ptr, rows, cols, pitch


def _out_step(code: int, out_scale) -> float:
    if code == _abi.INT8:
        if out_scale is None:
            raise ValueError("an int8 result needs out_scale, what one of its steps is worth")
        return float(out_scale)
    if out_scale is not None:
        raise ValueError("out_scale belongs to an int8 result")
    return 0.0


def _describe(m, k, lda, n, bk, ldb, y, row_scale, col_scale, bias, activation, residual, out_scale,
              groups, device):
    """(packed int8conv_matmul, address of y)."""
    if bk != k:
        raise ValueError(f"a has {k} columns, b has {bk}")
    y_ptr, ym, yn, ldy = _matrix("y", y, device)
    if ym != m or yn != n:
        _fail("y", f"a {m} x {n} matrix", y)
    dtype = y.dtype
    code = _dtype_code(dtype)
    res_ptr = ldr = 0
    if residual is not None:
        if residual.dtype != dtype:
            _fail("residual", f"a {dtype} matrix, like y", residual)
        res_ptr, rm, rn, ldr = _matrix("residual", residual, device)
        if rm != m or rn != n:
            _fail("residual", f"a {m} x {n} matrix", residual)
    return _pack(_MATMUL, m, n, k, lda, ldb, ldy, ldr,
                 _vector("row_scale", row_scale, m, device),
                 _vector("col_scale", col_scale, n * groups, device),
                 _vector("bias", bias, n * groups, device), res_ptr,
                 _activation(activation), code, _out_step(code, out_scale)), y_ptr


def launch_matmul(a, b, y, *, row_scale=None, col_scale=None, bias=None, activation: str = "none",
                  residual=None, out_scale=None, stream=None) -> None:
    """int8conv_launch_matmul: y = act(a @ b.T * row_scale * col_scale + bias) + residual.

    `a` int8 [m, k], `b` int8 [n, k]; `y` [m, n] in bfloat16, float16, float32,
    or int8 with `out_scale` (then without residual); `row_scale` [m],
    `col_scale` [n] and `bias` [n] float32, each optional; `residual` like `y`
    (it may be `y`).  The sums are exact, the epilogue is fp32 and rounds once."""
    device = _device_index()
    if stream is None and _calls is not None and y is not None and _calls.matmul(
            a, b, None, y, row_scale, col_scale, bias, residual, _activation(activation), 0,
            out_scale) is not None:
        return
    bp, n, bk, ldb = _int8_matrix("b", b, device)
    ap, m, k, lda = _int8_matrix("a", a, device)
    d, yp = _describe(m, k, lda, n, bk, ldb, y, row_scale, col_scale, bias, activation, residual,
                      out_scale, 1, device)
    status = _abi.lib.int8conv_launch_matmul(d, ap, bp, yp, _stream_handle(stream, device))
    if status:
        _abi.check(status, "matmul")


def launch_grouped_matmul(a, b, offsets, y, *, row_scale=None, col_scale=None, bias=None,
                          activation: str = "none", out_scale=None, stream=None) -> None:
    """int8conv_launch_grouped_matmul: rows offsets[e] .. offsets[e+1]-1 of `a`
    times b[e].T, for every expert e.

    `a` int8 [m, k] sorted by expert; `b` int8 [experts, n, k]; `offsets` int32
    [experts + 1] on the device, ascending; `col_scale` and `bias` [experts, n].
    Rows of `y` outside [offsets[0], offsets[experts]) are left as they were."""
    device = _device_index()
    if offsets is None:
        _fail("offsets", "an int32 tensor", None)
    if stream is None and _calls is not None and y is not None and _calls.matmul(
            a, b, offsets, y, row_scale, col_scale, bias, None, _activation(activation), 0,
            out_scale) is not None:
        return
    shape = b.shape
    if len(shape) != 3 or b.dtype != _torch.int8:
        _fail("b", "an int8 tensor [experts, n, k]", b)
    groups, n, bk = shape
    if not 1 <= groups <= 1024:
        raise ValueError(f"b: expected 1 to 1024 experts, got {groups}")
    group_stride, ldb, unit = b.stride()
    if unit != 1 and bk > 1:
        _fail("b", "a tensor whose last dimension is adjacent", b)
    if n <= 1:
        ldb = (bk + 15) & -16
    if ldb < bk or ldb & 15 or (groups > 1 and (group_stride & 15
                                                or group_stride < (n - 1) * ldb + bk)):
        _fail("b", "rows and experts that do not overlap, multiples of 16 bytes apart", b)
    if groups == 1:
        group_stride = 0
    if b.get_device() != device:
        _misplaced("b", b, device)
    ap, m, k, lda = _int8_matrix("a", a, device)
    d, yp = _describe(m, k, lda, n, bk, ldb, y, row_scale, col_scale, bias, activation, None,
                      out_scale, groups, device)
    status = _abi.lib.int8conv_launch_grouped_matmul(
        d, ap, b.data_ptr(), group_stride,
        _vector("offsets", offsets, groups + 1, device, _torch.int32), groups, yp,
        _stream_handle(stream, device))
    if status:
        _abi.check(status, "grouped_matmul")


def _empty(shape, dtype, like, stream):
    """An uninitialised tensor on `like`'s device, allocated on the launch's
    stream, so that what a call frees on return is reused in that stream's
    order.  int8 rows get a pitch that is a multiple of 16."""
    torch = _torch or _load_torch()
    if stream is not None:
        if isinstance(stream, int):
            stream = torch.cuda.ExternalStream(stream)
        with torch.cuda.stream(stream):
            return _empty(shape, dtype, like, None)
    if dtype == torch.int8 and shape[-1] & 15:
        cols = shape[-1]
        return like.new_empty((*shape[:-1], (cols + 15) & -16), dtype=dtype)[..., :cols]
    return like.new_empty(shape, dtype=dtype)


def matmul(a, b, *, row_scale=None, col_scale=None, bias=None, activation: str = "none",
           residual=None, dtype=None, out_scale=None, stream=None):
    """launch_matmul into a new result of type `dtype` (default: the residual's
    type, else bfloat16)."""
    torch = _torch or _load_torch()
    if dtype is None:
        dtype = residual.dtype if residual is not None else torch.bfloat16
    if stream is None and _calls is not None:
        y = _calls.matmul(a, b, None, None, row_scale, col_scale, bias, residual,
                          _activation(activation), _dtype_code(dtype), out_scale)
        if y is not None:
            return y
    y = _empty((a.shape[0], b.shape[0]), dtype, a, stream)
    launch_matmul(a, b, y, row_scale=row_scale, col_scale=col_scale, bias=bias,
                  activation=activation, residual=residual, out_scale=out_scale, stream=stream)
    return y


def grouped_matmul(a, b, offsets, *, row_scale=None, col_scale=None, bias=None,
                   activation: str = "none", dtype=None, out_scale=None, stream=None):
    """launch_grouped_matmul into a new result of type `dtype` (default
    bfloat16); rows that belong to no expert are uninitialised."""
    torch = _torch or _load_torch()
    if dtype is None:
        dtype = torch.bfloat16
    if offsets is None:
        _fail("offsets", "an int32 tensor", None)
    if stream is None and _calls is not None:
        y = _calls.matmul(a, b, offsets, None, row_scale, col_scale, bias, None,
                          _activation(activation), _dtype_code(dtype), out_scale)
        if y is not None:
            return y
    if len(b.shape) != 3:
        _fail("b", "an int8 tensor [experts, n, k]", b)
    y = _empty((a.shape[0], b.shape[1]), dtype, a, stream)
    launch_grouped_matmul(a, b, offsets, y, row_scale=row_scale, col_scale=col_scale, bias=bias,
                          activation=activation, out_scale=out_scale, stream=stream)
    return y


def launch_quantize_rows(x, q, scale, index=None, *, stream=None) -> None:
    """int8conv_launch_quantize_rows: scale[i] = max|x[r]| / 127 and
    q[i] = round(x[r] / scale[i]), r = index[i] (or i without `index`).

    `x` [rows, k] in bfloat16, float16 or float32; `q` int8 [m, k]; `scale`
    float32 [m]; `index` int32 [m] on the device.  A row with an infinity or a
    NaN gets scale NaN and zeros; an index outside [0, rows) scale 0 and zeros."""
    device = _device_index()
    if stream is None and _calls is not None and q is not None and _calls.quantize_rows(
            x, index, q, scale) is not None:
        return
    x_ptr, rows, k, ldx = _matrix("x", x, device)
    code = _dtype_code(x.dtype)
    if q.dtype != _torch.int8:
        _fail("q", "an int8 matrix", q)
    q_ptr, m, qk, ldq = _matrix("q", q, device)
    if qk != k:
        _fail("q", f"{k} columns, like x", q)
    if index is None and rows != m:
        _fail("q", f"{rows} rows, like x", q)
    if scale is None:
        _fail("scale", "a float32 tensor", None)
    status = _abi.lib.int8conv_launch_quantize_rows(
        m, k, code, x_ptr, rows, ldx, _vector("index", index, m, device, _torch.int32), q_ptr, ldq,
        _vector("scale", scale, m, device), _stream_handle(stream, device))
    if status:
        _abi.check(status, "quantize_rows")


def quantize_rows(x, index=None, *, stream=None):
    """launch_quantize_rows into new buffers: (q, scale).  With `index`, row i of
    the result is x[index[i]]: the gather of an expert dispatch."""
    torch = _torch or _load_torch()
    if stream is None and _calls is not None:
        pair = _calls.quantize_rows(x, index, None, None)
        if pair is not None:
            return pair
    shape = x.shape
    if len(shape) != 2:
        _fail("x", "a matrix", x)
    m = shape[0] if index is None else index.numel()
    q = _empty((m, shape[1]), torch.int8, x, stream)
    scale = _empty((m,), torch.float32, x, stream)
    launch_quantize_rows(x, q, scale, index, stream=stream)
    return q, scale


def _pixels(name: str, t, device: int):
    """(address, images, positions, channels, pitch) of a channels-last tensor
    [n, ..., c] whose positions are evenly spaced."""
    shape, strides = t.shape, t.stride()
    if len(shape) < 2 or (strides[-1] != 1 and shape[-1] > 1):
        _fail(name, "a channels-last tensor [n, ..., c]", t)
    if t.get_device() != device:
        _misplaced(name, t, device)
    n, c = shape[0], shape[-1]
    positions, pitch = 1, None
    for i in range(len(shape) - 2, -1, -1):
        size = shape[i]
        if size > 1:
            if pitch is None:
                pitch = strides[i]
            elif strides[i] != pitch * positions:
                _fail(name, "evenly spaced positions", t)
        positions *= size
    if pitch is None:
        pitch = c
    elif pitch < c:
        _fail(name, "positions that do not overlap", t)
    return t.data_ptr(), n, positions // n if n else 0, c, pitch


def _norm_desc(x, groups, y, gamma, beta, eps, activation, scale, out_scale, device):
    """(packed int8conv_group_norm, addresses of x and y)."""
    x_ptr, n, pixels, c, ldx = _pixels("x", x, device)
    if y.shape != x.shape:
        _fail("y", f"a tensor of shape {tuple(x.shape)}", y)
    y_ptr, _, _, _, ldy = _pixels("y", y, device)
    code = _dtype_code(y.dtype)
    return _pack(_NORM, n, pixels, c, int(groups), ldx, ldy, _vector("scale", scale, c, device),
                 _vector("gamma", gamma, c, device), _vector("beta", beta, c, device),
                 float(eps), _activation(activation), _dtype_code(x.dtype), code,
                 _out_step(code, out_scale)), x_ptr, y_ptr


def group_norm_workspace_bytes(x, groups: int, y) -> int:
    """Bytes of scratch that launch_group_norm(x, groups, y, ...) needs."""
    device = _device_index()
    d, _, _ = _norm_desc(x, groups, y, None, None, 1e-5, "none", None,
                         1.0 if y.dtype == _torch.int8 else None, device)
    return _abi.lib.int8conv_group_norm_workspace_bytes(d)


def launch_group_norm(x, groups: int, y, gamma=None, beta=None, *, eps: float = 1e-5,
                      activation: str = "none", scale=None, out_scale=None, workspace=None,
                      workspace_bytes: int = 0, stream=None) -> None:
    """int8conv_launch_group_norm: y = act(norm(x * scale) * gamma + beta), statistics
    over each image's positions and each group's channels.

    `x` [n, ..., c] in bfloat16, float16, float32 or int32 (a convolution's
    output, `scale` [c] what one step of each channel is worth); `y` of the same
    shape in bfloat16, float16, float32, or int8 with `out_scale`; `gamma`,
    `beta`, `scale` float32 [c], each optional; `workspace` at least
    group_norm_workspace_bytes() on the device, one for each launch that may run
    at the same time."""
    device = _device_index()
    d, x_ptr, y_ptr = _norm_desc(x, groups, y, gamma, beta, eps, activation, scale, out_scale,
                                 device)
    ws = 0
    if workspace is not None:
        if isinstance(workspace, int):
            ws = workspace
        else:
            if workspace.get_device() != device:
                _misplaced("workspace", workspace, device)
            size = workspace.numel() * workspace.element_size()
            if not workspace.is_contiguous() or workspace_bytes > size:
                _fail("workspace", f"{workspace_bytes} contiguous bytes", workspace)
            ws = workspace.data_ptr()
    status = _abi.lib.int8conv_launch_group_norm(d, x_ptr, y_ptr, ws, int(workspace_bytes),
                                                 _stream_handle(stream, device))
    if status:
        _abi.check(status, "group_norm")


def group_norm(x, groups: int, gamma=None, beta=None, *, eps: float = 1e-5,
               activation: str = "none", scale=None, dtype=None, out_scale=None, stream=None):
    """launch_group_norm into a new result of type `dtype` (default: x's type, or
    bfloat16 for int32).  An int8 result has its positions a multiple of 16 bytes
    apart, as the convolution and the products read them."""
    device = _device_index()
    if dtype is None:
        dtype = _torch.bfloat16 if x.dtype == _torch.int32 else x.dtype
    if stream is None and _calls is not None:
        y = _calls.group_norm(x, groups, gamma, beta, scale, eps, _activation(activation),
                              _dtype_code(dtype), out_scale)
        if y is not None:
            return y
    y = _empty(x.shape, dtype, x, stream)
    d, x_ptr, y_ptr = _norm_desc(x, groups, y, gamma, beta, eps, activation, scale, out_scale,
                                 device)
    nbytes = _abi.lib.int8conv_group_norm_workspace_bytes(d)
    ws = _empty((nbytes,), _torch.uint8, x, stream) if nbytes else None
    status = _abi.lib.int8conv_launch_group_norm(d, x_ptr, y_ptr,
                                                 0 if ws is None else ws.data_ptr(), nbytes,
                                                 _stream_handle(stream, device))
    if status:
        _abi.check(status, "group_norm")
    return y
