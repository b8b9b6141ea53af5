"""Products, row quantisation and group norm on CUDA tensors: what an int8
model runs between its convolutions (no reference counterpart).

    q, row = quantize_rows(x)                    # [m, k] floats -> int8, a scale per row
    y = matmul(q, w, row_scale=row, col_scale=col, bias=b, activation="silu", residual=r)
    y = grouped_matmul(q, experts, offsets, row_scale=row, col_scale=cols)
    z = group_norm(acc, 32, gamma, beta, scale=s, activation="silu", dtype=torch.int8, out_scale=t)

`launch_*` write into the caller's buffers and never allocate; the plain names
allocate the result (and the group norm's workspace) on the launch's stream.
Everything is asynchronous on `stream` (default: the current one), runs on the
current CUDA device and may be captured into a graph.  Wrong arguments raise
ValueError (types, sizes, devices) or Int8ConvError (the library's own checks).

int8 matrices are rows of k bytes whose pitch is a multiple of 16 (the copies
into shared memory move 16-byte units): the int8 results here come that way, as
views of wider rows where k is not a multiple of 16.  A weight matrix [n, k] in
floats becomes such a matrix, with a scale per output channel, through
quantize_rows too.
"""
from __future__ import annotations

from ctypes import byref

from . import _abi
from .api import _stream


def _fail(name: str, want: str, t) -> None:
    if t is None:
        raise ValueError(f"{name}: expected {want}, got None")
    raise ValueError(f"{name}: expected {want}, got {t.dtype} {tuple(t.shape)} with strides "
                     f"{tuple(t.stride())} on {t.device}")


_DTYPES: dict = {}


def _dtype_code(dtype) -> int:
    if not _DTYPES:
        import torch

        _DTYPES.update({getattr(torch, name): code for name, code in _abi.DTYPES.items()})
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"unsupported type {dtype}")
    return code


def _activation(name: str) -> int:
    code = _abi.ACTIVATIONS.get(name)
    if code is None:
        raise ValueError(f"activation: expected one of {sorted(_abi.ACTIVATIONS)}, got {name!r}")
    return code


def _device_index() -> int:
    import torch

    return torch.cuda.current_device()


def _on(name: str, t, device: int) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor, got one on {t.device}")
    if t.device.index != device:
        raise ValueError(f"{name} on {t.device}, but the current CUDA device is cuda:{device}: "
                         f"launch under torch.cuda.device({t.device.index}) or move the buffers")


def _vector(name: str, t, count: int, device: int, dtype=None) -> int:
    """Address of an optional contiguous fp32 vector of `count` entries."""
    if t is None:
        return 0
    import torch

    if t.dtype != (dtype or torch.float32) or t.numel() != count or not t.is_contiguous():
        _fail(name, f"a contiguous {dtype or torch.float32} tensor of {count} elements", t)
    _on(name, t, device)
    return t.data_ptr()


def _matrix(name: str, t, device: int):
    """(address, rows, columns, pitch) of a matrix with adjacent columns."""
    if t.dim() != 2 or (t.stride(1) != 1 and t.shape[1] > 1):
        _fail(name, "a matrix whose columns are adjacent", t)
    _on(name, t, device)
    rows, cols = t.shape
    # One row has no pitch of its own.
    pitch = t.stride(0) if rows > 1 else cols
    if pitch < cols:
        _fail(name, "rows that do not overlap", t)
    return t.data_ptr(), rows, cols, pitch


def _int8_matrix(name: str, t, device: int):
    import torch

    if t.dtype != torch.int8:
        _fail(name, "an int8 matrix", t)
    ptr, rows, cols, pitch = _matrix(name, t, device)
    if rows <= 1:
        pitch = (cols + 15) // 16 * 16
    elif pitch % 16:
        raise ValueError(f"{name}: rows are {pitch} bytes apart, which is not a multiple of 16 "
                         "(quantize_rows returns rows that are)")
    return ptr, rows, cols, pitch


def _describe(a, b_shape, y, row_scale, col_scale, bias, activation, residual, out_scale, groups,
              device):
    a_ptr, m, k, lda = a
    n, bk, ldb = b_shape
    if bk != k:
        raise ValueError(f"a has {k} columns, b has {bk}")
    y_ptr, ym, yn, ldy = _matrix("y", y, device)
    if (ym, yn) != (m, n):
        _fail("y", f"a {m} x {n} matrix", y)
    d = _abi.CMatmul()
    d.m, d.n, d.k, d.lda, d.ldb, d.ldy = m, n, k, lda, ldb, ldy
    d.y_dtype = _dtype_code(y.dtype)
    d.activation = _activation(activation)
    d.row_scale = _vector("row_scale", row_scale, m, device)
    d.col_scale = _vector("col_scale", col_scale, n * groups, device)
    d.bias = _vector("bias", bias, n * groups, device)
    if residual is not None:
        if residual.dtype != y.dtype:
            _fail("residual", f"a {y.dtype} matrix, like y", residual)
        d.residual, rm, rn, d.ldr = _matrix("residual", residual, device)
        if (rm, rn) != (m, n):
            _fail("residual", f"a {m} x {n} matrix", residual)
    if d.y_dtype == _abi.INT8:
        if out_scale is None:
            raise ValueError("an int8 result needs out_scale, what one of its steps is worth")
        d.out_scale = float(out_scale)
    elif out_scale is not None:
        raise ValueError("out_scale belongs to an int8 result")
    return d, y_ptr


def launch_matmul(a, b, y, *, row_scale=None, col_scale=None, bias=None, activation: str = "none",
                  residual=None, out_scale=None, stream=None) -> None:
    """int8conv_launch_matmul: y = act(a @ b.T * row_scale * col_scale + bias) + residual.

    `a` int8 [m, k], `b` int8 [n, k]; `y` [m, n] in bfloat16, float16, float32,
    or int8 with `out_scale` (then without residual); `row_scale` [m],
    `col_scale` [n] and `bias` [n] float32, each optional; `residual` like `y`
    (it may be `y`).  The sums are exact, the epilogue is fp32 and rounds once."""
    device = _device_index()
    bp, n, bk, ldb = _int8_matrix("b", b, device)
    am = _int8_matrix("a", a, device)
    d, y_ptr = _describe(am, (n, bk, ldb), y, row_scale, col_scale, bias, activation, residual,
                         out_scale, 1, device)
    _abi.check(_abi.lib.int8conv_launch_matmul(byref(d), am[0], bp, y_ptr, _stream(stream)),
               "matmul")


def launch_grouped_matmul(a, b, offsets, y, *, row_scale=None, col_scale=None, bias=None,
                          activation: str = "none", out_scale=None, stream=None) -> None:
    """int8conv_launch_grouped_matmul: rows offsets[e] .. offsets[e+1]-1 of `a`
    times b[e].T, for every expert e.

    `a` int8 [m, k] sorted by expert; `b` int8 [experts, n, k]; `offsets` int32
    [experts + 1] on the device, ascending; `col_scale` and `bias` [experts, n].
    Rows of `y` outside [offsets[0], offsets[experts]) are left as they were."""
    import torch

    device = _device_index()
    if b.dim() != 3 or b.dtype != torch.int8:
        _fail("b", "an int8 tensor [experts, n, k]", b)
    groups = b.shape[0]
    if not 1 <= groups <= 1024:
        raise ValueError(f"b: expected 1 to 1024 experts, got {groups}")
    bp, n, bk, ldb = _int8_matrix("b", b[0], device)
    group_stride = b.stride(0) if groups > 1 else 0
    if groups > 1 and (group_stride % 16 or group_stride < (n - 1) * ldb + bk):
        _fail("b", "experts that do not overlap, a multiple of 16 bytes apart", b)
    am = _int8_matrix("a", a, device)
    d, y_ptr = _describe(am, (n, bk, ldb), y, row_scale, col_scale, bias, activation, None,
                         out_scale, groups, device)
    o = _vector("offsets", offsets, groups + 1, device, torch.int32)
    if not o:
        raise ValueError("offsets: expected an int32 tensor, got None")
    _abi.check(_abi.lib.int8conv_launch_grouped_matmul(byref(d), am[0], bp, group_stride, o, groups,
                                                       y_ptr, _stream(stream)), "grouped_matmul")


def _int8_rows(rows: int, cols: int, device):
    """An uninitialised int8 matrix whose pitch is a multiple of 16."""
    import torch

    pitch = (cols + 15) // 16 * 16
    t = torch.empty((rows, pitch), dtype=torch.int8, device=device)
    return t if pitch == cols else t[:, :cols]


class _Allocating:
    """Allocates on the launch's stream, so that what a call frees on return is
    reused in that stream's order."""

    def __init__(self, stream):
        import torch

        self.guard = None
        if stream is not None:
            if isinstance(stream, int):
                stream = torch.cuda.ExternalStream(stream)
            self.guard = torch.cuda.stream(stream)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _result(m: int, n: int, dtype, device, stream):
    import torch

    with _Allocating(stream):
        if dtype == torch.int8:
            return _int8_rows(m, n, device)
        return torch.empty((m, n), dtype=dtype, device=device)


def matmul(a, b, *, row_scale=None, col_scale=None, bias=None, activation: str = "none",
           residual=None, dtype=None, out_scale=None, stream=None):
    """launch_matmul into a new result of type `dtype` (default: the residual's
    type, else bfloat16)."""
    import torch

    if dtype is None:
        dtype = residual.dtype if residual is not None else torch.bfloat16
    y = _result(a.shape[0], b.shape[0], dtype, a.device, stream)
    launch_matmul(a, b, y, row_scale=row_scale, col_scale=col_scale, bias=bias,
                  activation=activation, residual=residual, out_scale=out_scale, stream=stream)
    return y


def grouped_matmul(a, b, offsets, *, row_scale=None, col_scale=None, bias=None,
                   activation: str = "none", dtype=None, out_scale=None, stream=None):
    """launch_grouped_matmul into a new result of type `dtype` (default
    bfloat16); rows that belong to no expert are uninitialised."""
    import torch

    y = _result(a.shape[0], b.shape[1], dtype or torch.bfloat16, a.device, stream)
    launch_grouped_matmul(a, b, offsets, y, row_scale=row_scale, col_scale=col_scale, bias=bias,
                          activation=activation, out_scale=out_scale, stream=stream)
    return y


def launch_quantize_rows(x, q, scale, index=None, *, stream=None) -> None:
    """int8conv_launch_quantize_rows: scale[i] = max|x[r]| / 127 and
    q[i] = round(x[r] / scale[i]), r = index[i] (or i without `index`).

    `x` [rows, k] in bfloat16, float16 or float32; `q` int8 [m, k]; `scale`
    float32 [m]; `index` int32 [m] on the device.  A row with an infinity or a
    NaN gets scale NaN and zeros; an index outside [0, rows) scale 0 and zeros."""
    import torch

    device = _device_index()
    x_ptr, rows, k, ldx = _matrix("x", x, device)
    code = _dtype_code(x.dtype)
    if q.dtype != torch.int8:
        _fail("q", "an int8 matrix", q)
    q_ptr, m, qk, ldq = _matrix("q", q, device)
    if qk != k:
        _fail("q", f"{k} columns, like x", q)
    index_ptr = _vector("index", index, m, device, torch.int32)
    if index is None and rows != m:
        _fail("q", f"{rows} rows, like x", q)
    scale_ptr = _vector("scale", scale, m, device)
    _abi.check(_abi.lib.int8conv_launch_quantize_rows(
        m, k, code, x_ptr, rows, ldx, index_ptr or None, q_ptr, ldq, scale_ptr, _stream(stream)),
        "quantize_rows")


def quantize_rows(x, index=None, *, stream=None):
    """launch_quantize_rows into new buffers: (q, scale).  With `index`, row i of
    the result is x[index[i]]: the gather of an expert dispatch."""
    import torch

    m = x.shape[0] if index is None else index.numel()
    if x.dim() != 2:
        _fail("x", "a matrix", x)
    with _Allocating(stream):
        q = _int8_rows(m, x.shape[1], x.device)
        scale = torch.empty(m, dtype=torch.float32, device=x.device)
    launch_quantize_rows(x, q, scale, index, stream=stream)
    return q, scale


def _pixels(name: str, t, device: int):
    """(address, images, positions, channels, pitch) of a channels-last tensor
    [n, ..., c] whose positions are evenly spaced."""
    if t.dim() < 2 or (t.stride(-1) != 1 and t.shape[-1] > 1):
        _fail(name, "a channels-last tensor [n, ..., c]", t)
    _on(name, t, device)
    shape, strides = t.shape, t.stride()
    c, positions, pitch = shape[-1], 1, None
    for size, stride in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if size > 1:
            if pitch is None:
                pitch = stride
            elif stride != pitch * positions and t.numel():
                _fail(name, "evenly spaced positions", t)
        positions *= size
    n = shape[0]
    pitch = c if pitch is None else pitch
    if pitch < c:
        _fail(name, "positions that do not overlap", t)
    pixels = 1
    for size in shape[1:-1]:
        pixels *= size
    return t.data_ptr(), n, pixels, c, pitch


def _norm_desc(x, groups, y, gamma, beta, eps, activation, scale, out_scale, device):
    x_ptr, n, pixels, c, ldx = _pixels("x", x, device)
    if tuple(y.shape) != tuple(x.shape):
        _fail("y", f"a tensor of shape {tuple(x.shape)}", y)
    y_ptr, _, _, _, ldy = _pixels("y", y, device)
    d = _abi.CGroupNorm()
    d.n, d.pixels, d.channels, d.groups, d.ldx, d.ldy = n, pixels, c, int(groups), ldx, ldy
    d.scale = _vector("scale", scale, c, device)
    d.gamma = _vector("gamma", gamma, c, device)
    d.beta = _vector("beta", beta, c, device)
    d.eps = float(eps)
    d.activation = _activation(activation)
    d.x_dtype, d.y_dtype = _dtype_code(x.dtype), _dtype_code(y.dtype)
    if d.y_dtype == _abi.INT8:
        if out_scale is None:
            raise ValueError("an int8 result needs out_scale, what one of its steps is worth")
        d.out_scale = float(out_scale)
    elif out_scale is not None:
        raise ValueError("out_scale belongs to an int8 result")
    return d, x_ptr, y_ptr


def group_norm_workspace_bytes(x, groups: int, y) -> int:
    """Bytes of scratch that launch_group_norm(x, groups, y, ...) needs."""
    d, _, _ = _norm_desc(x, groups, y, None, None, 1e-5, "none", None,
                         1.0 if _dtype_code(y.dtype) == _abi.INT8 else None, _device_index())
    return int(_abi.lib.int8conv_group_norm_workspace_bytes(byref(d)))


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
        if not isinstance(workspace, int):
            _on("workspace", workspace, device)
            size = workspace.numel() * workspace.element_size()
            if not workspace.is_contiguous() or workspace_bytes > size:
                _fail("workspace", f"{workspace_bytes} contiguous bytes", workspace)
            workspace = workspace.data_ptr()
        ws = workspace
    _abi.check(_abi.lib.int8conv_launch_group_norm(byref(d), x_ptr, y_ptr, ws, int(workspace_bytes),
                                                   _stream(stream)), "group_norm")


def group_norm(x, groups: int, gamma=None, beta=None, *, eps: float = 1e-5,
               activation: str = "none", scale=None, dtype=None, out_scale=None, stream=None):
    """launch_group_norm into a new result of type `dtype` (default: x's type, or
    bfloat16 for int32).  An int8 result has its positions a multiple of 16 bytes
    apart, as the convolution and the products read them."""
    import torch

    if dtype is None:
        dtype = torch.bfloat16 if x.dtype == torch.int32 else x.dtype
    device = _device_index()
    with _Allocating(stream):
        if dtype == torch.int8 and x.dim() >= 2:
            c = x.shape[-1]
            y = torch.empty((*x.shape[:-1], (c + 15) // 16 * 16), dtype=dtype,
                            device=x.device)[..., :c]
        else:
            y = torch.empty(x.shape, dtype=dtype, device=x.device)
        d, x_ptr, y_ptr = _norm_desc(x, groups, y, gamma, beta, eps, activation, scale, out_scale,
                                     device)
        nbytes = int(_abi.lib.int8conv_group_norm_workspace_bytes(byref(d)))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
    _abi.check(_abi.lib.int8conv_launch_group_norm(byref(d), x_ptr, y_ptr,
                                                   0 if ws is None else ws.data_ptr(), nbytes,
                                                   _stream(stream)), "group_norm")
    return y
