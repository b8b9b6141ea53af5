"""Plain 64-bit forms of the products, the row quantisation and the group norm,
with the error that the kernels' fp32 arithmetic and one rounding may add.

Units: u = 2^-24 is half an fp32 step relative to the value.
"""
import math

import torch

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U}
# Half a step below the smallest normal number, where steps stop shrinking.
FLOOR = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def act(v, name):
    if name == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v / math.sqrt(2)))
    if name == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    if name == "silu":
        return v * torch.sigmoid(v)
    return v


def act_error(v, err, name):
    """Error of an activation of v whose argument is off by err: no slope passes
    1.13; the approximate exponential and quotient are off by 2^-19, erf by a
    few units relative to |v|."""
    if name in ("none", "relu"):
        return err
    return 1.13 * err + 2.0 ** -19 * v.abs()


def check(got, want, err, what=""):
    """got: what the kernel wrote; want: fp64; err: fp64 error before the rounding."""
    got64 = got.double().cpu()
    tol = err + (want.abs() + err) * HALF[got.dtype] + FLOOR[got.dtype]
    both_nan = torch.isnan(want) & torch.isnan(got64)
    ok = both_nan | (got64 == want) | ((got64 - want).abs() <= tol)
    if not bool(ok.all()):
        i = int((~ok).flatten().nonzero()[0])
        raise AssertionError(f"{what}: {int((~ok).sum())} of {ok.numel()} off, first at {i}: got "
                             f"{got64.flatten()[i]}, want {want.flatten()[i]} +- {tol.flatten()[i]}")


def check_int8(got, want, err, what=""):
    """want: the value in steps, before clamping and rounding."""
    got64 = got.double().cpu()
    lo, hi = want - err - 0.5, want + err + 0.5
    ok = (got64 >= lo.clamp(-128, 127)) & (got64 <= hi.clamp(-128, 127))
    ok |= torch.isnan(want) & (got64 == 0)
    assert bool(ok.all()), f"{what}: {int((~ok).sum())} of {ok.numel()} off"


def product(a, b, row=None, col=None, bias=None, activation="none", residual=None):
    """(value, error) of one product.  The integer sum becomes fp32 (u), is
    multiplied by the column scale (u) and then by the row scale with the bias
    added (u of the sum); the residual's sum is one more."""
    p = a.double().cpu() @ b.double().cpu().t()
    if col is not None:
        p = p * col.double().cpu()
    if row is not None:
        p = p * row.double().cpu()[:, None]
    v = p if bias is None else p + bias.double().cpu()
    err = act_error(v, U * (2.01 * p.abs() + 1.01 * v.abs()), activation)
    y = act(v, activation)
    if residual is not None:
        y = y + residual.double().cpu()
        err = err + 1.01 * U * y.abs()
    return y, err


def quantized(x):
    """(q, scale) by the formula's own fp32 arithmetic, on the CPU: IEEE division
    and rounding to even leave one answer, bit for bit."""
    x = x.float().cpu()
    scale = x.abs().amax(1) / 127 if x.shape[1] else torch.zeros(x.shape[0])
    bad = ~torch.isfinite(x).all(1)
    scale[bad] = float("nan")
    ok = (scale > 0)[:, None]
    q = torch.where(ok, torch.round(x / torch.where(ok, scale[:, None], 1.0)), 0.0)
    return torch.nan_to_num(q).clamp(-127, 127).to(torch.int8), scale


def norm(x, groups, gamma=None, beta=None, eps=1e-5, activation="none", scale=None, terms=64):
    """(value, error) of a group norm of x [n, p, c].

    `terms`: the longest run of additions one thread makes, plus the joins.  A
    sum of that many terms is off by at most terms * u relative to the sum of
    magnitudes, so the mean by terms * u * (mean |v - shift| + |mean| / terms):
    with a shift from the data, deviations D = max |v - mean| bound it by
    2 * terms * u * D + u * |mean|.  The variance is off by 4 * terms * u of
    itself plus that of the mean's error squared; v itself by u * |v|."""
    x = x.double().cpu()
    n, p, c = x.shape
    if scale is not None:
        x = x * scale.double().cpu()
    v = x.reshape(n, p, groups, c // groups)
    mean = v.mean((1, 3), keepdim=True)
    dev = v - mean
    var = (dev * dev).mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    z = dev * rstd
    far = dev.abs().amax((1, 3), keepdim=True)
    merr = U * (2 * terms * far + 4 * (mean.abs() + far))
    # A thread's squares are taken about its shift, up to 2 far away.
    verr = 4 * terms * U * (var + far * far / max(1, p)) + merr * merr + 8 * U * far * far
    rel = 0.5 * verr * rstd * rstd + 4 * U
    err = (merr + 2 * U * v.abs()) * rstd + z.abs() * rel
    z, err = z.reshape(n, p, c), err.expand_as(z).reshape(n, p, c)
    w = torch.ones(c, dtype=torch.float64) if gamma is None else gamma.double().cpu()
    b = torch.zeros(c, dtype=torch.float64) if beta is None else beta.double().cpu()
    y = z * w + b
    err = err * w.abs() + U * (2 * (z * w).abs() + 2 * y.abs())
    return act(y, activation), act_error(y, err, activation)
