"""The group norm's statistics where a few positions lie far from the others:
the corner of a zero-padded image, a first token with massive activations."""
import pytest
import torch

import int8_kernel_lab_b200 as m
from operators_reference import HALF, U

pytestmark = pytest.mark.gpu


def _exact(x, groups, scale=None):
    """(normalised values, mean / deviation) of one image [p, c] in 64 bits, on the GPU."""
    v = x.double()
    if scale is not None:
        v = v * scale.double()
    p, c = v.shape
    v = v.view(p, groups, c // groups)
    var, mean = torch.var_mean(v, dim=(0, 2), unbiased=False, keepdim=True)
    rstd = 1 / (var + 1e-5).sqrt()
    return ((v - mean) * rstd).view(p, c), (mean.abs() * rstd).expand_as(v).reshape(p, c), \
        (v.abs() * rstd).reshape(p, c)


def _tolerance(z, mean, size, p, c, vec):
    """Half an fp32 step is u.  A run of a thread is at most 128 positions.

    Variance: adding the k-th of n squares about a shift that is the mean of m of
    them costs u times a sum of at most n / m times what they come to, on average
    half of it.  A thread with up to 24 positions: 24 * 24 / 2.  With more: 8 * 8 / 2
    up to 8, 24 * 4 / 2 up to 32, 96 * 2 / 2 up to the first run, 128 in the runs
    and 2 for each; all below 2 * (128 + runs) + 64.  Then up to `lanes`
    threads of a column, 32 steps over channels and CTAs.  Half of the relative
    error reaches 1 / deviation.
    Mean, in deviations: a run's sum starts near zero, so 128 steps of the
    values' mean distance (below 1.5 deviations, 200 in all); the threads' means
    relative to the first one's, which may be sqrt(lanes) deviations away, over
    `lanes` steps; the mean's own rounding, and its use in the input's units.
    Each value times its scale, and the formula's own four roundings, come on top."""
    lanes = 512 // min(512, c // 8 if vec else c)
    chain = 2 * (128 + p / (32 * lanes) + 1) + 64 + lanes + 32
    return U * (z.abs() * (chain / 2 + 4) + 200 + lanes ** 1.5 + 4 * mean + 4 * size)


def _check(x, groups, scale=None):
    n, p, c = x.shape
    y = m.group_norm(x, groups, scale=scale, dtype=torch.float32)
    for i in range(n):
        z, mean, size = _exact(x[i], groups, scale)
        off = (y[i].double() - z).abs()
        tol = _tolerance(z, mean, size, p, c, c % 8 == 0)
        worst = float((off / tol).max())
        assert worst <= 1, f"image {i}: {worst:.3g} of the tolerance"
    assert m.device_status() == 0


@pytest.mark.parametrize("far", [100.0, 10000.0, "padding"])
@pytest.mark.parametrize("n,p,c,groups", [
    (256, 3136, 256, 32),     # a CTA for each image
    (256, 4096, 260, 10),     # channel by channel, one thread down each
    (256, 4096, 258, 258),
    (40, 3000, 128, 4),       # clusters
    (4, 16384, 64, 8),        # chunks, two kernels
    (1, 200000, 8, 2),
    (3, 5, 64, 8),            # less than a batch for each thread
    (300, 70, 4096, 32),      # one thread down each column of 8 channels
], ids=str)
def test_first_position_far_from_the_others(cuda, n, p, c, groups, far):
    g = torch.Generator(device="cuda").manual_seed(60)
    x = torch.randn(n, p, c, generator=g, device="cuda")
    if far == "padding":
        x += 1000
        x[:, 0] = 0
    else:
        x[:, 0] = far
    _check(x, groups)


@pytest.mark.parametrize("at", [1, 37, 1500, 2999])
def test_far_position_anywhere(cuda, at):
    x = torch.randn(20, 3000, 72, generator=torch.Generator(device="cuda").manual_seed(61),
                    device="cuda")
    x[:, at] = -3000.0
    _check(x, 9)
    _check(x[..., :70].contiguous(), 7)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.int32], ids=str)
@pytest.mark.parametrize("n,p,c,groups", [(256, 3136, 128, 32), (8, 4096, 320, 32)], ids=str)
def test_far_first_position_of_other_types(cuda, dtype, n, p, c, groups):
    g = torch.Generator(device="cuda").manual_seed(62)
    x = torch.randn(n, p, c, generator=g, device="cuda") + 3
    x[:, 0] = 2000
    scale = None
    if dtype == torch.int32:
        scale = (torch.rand(c, generator=g, device="cuda") + 0.5) / 2000
        x = x * 2000
    _check(x.to(dtype), groups, scale)


def test_results_of_16_bits_are_rounded_once(cuda):
    x = torch.randn(256, 1000, 64, generator=torch.Generator(device="cuda").manual_seed(63),
                    device="cuda")
    x[:, 0] = 500
    y = m.group_norm(x, 8, dtype=torch.float16)
    for i in range(0, 256, 50):
        z, mean, size = _exact(x[i], 8)
        tol = _tolerance(z, mean, size, 1000, 64, True)
        tol = tol + (z.abs() + tol) * HALF[torch.float16] + 2.0 ** -25
        assert bool(((y[i].double() - z).abs() <= tol).all())


@pytest.mark.parametrize("n,p,c,groups", [(2, 90, 64, 8), (3, 4000, 40, 5), (1, 700, 30, 3)], ids=str)
@pytest.mark.parametrize("size", [1e-30, 1e-22, 1e22, 1e30])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_scale_makes_small_and_large_inputs_ordinary(cuda, dtype, size, n, p, c, groups):
    # The squares of x leave fp32's range, those of x * scale do not.
    g = torch.Generator(device="cuda").manual_seed(64)
    x = (torch.randn(n, p, c, generator=g, device="cuda") + 2).to(dtype)
    scale = torch.rand(c, generator=g, device="cuda") + 0.5
    scale[::3] /= size
    x[..., ::3] = (x[..., ::3].float() * size).to(dtype)
    _check(x, groups, scale)


def test_constant_channels_under_a_scale(cuda):
    # x * scale is rounded alike everywhere: the deviations are zero.
    x = torch.full((2, 500, 32), 12345.0, device="cuda")
    scale = torch.full((32,), 0.37, device="cuda")
    y = m.group_norm(x, 4, scale=scale, eps=1e-5)
    # The mean and its use in x's units are off by 2 u of the value, over sqrt(eps).
    assert float(y.abs().max()) <= 4 * U * 12345 * 0.37 / 1e-5 ** 0.5


@pytest.mark.parametrize("n,p,c,groups", [(2, 90, 64, 8), (3, 4000, 40, 5), (1, 700, 30, 3)], ids=str)
@pytest.mark.parametrize("small", [1e-30, -1e-32, 0.0])
def test_channel_far_smaller_than_its_group(cuda, small, n, p, c, groups):
    # The group's mean in the units of such a channel leaves fp32's range.
    g = torch.Generator(device="cuda").manual_seed(65)
    x = torch.randn(n, p, c, generator=g, device="cuda") * 1e8 + 1e9
    scale = torch.rand(c, generator=g, device="cuda") + 0.5
    scale[1::4] = small
    _check(x, groups, scale)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("n,p,c,groups,pitch", [
    (256, 400, 128, 8, 128),      # a CTA for each image
    (40, 3000, 128, 4, 136),      # clusters
    (8, 4096, 320, 32, 320),      # two kernels
    (30, 900, 70, 7, 75),         # channel by channel
    (2, 60000, 30, 3, 30),
    (1, 1, 48, 4, 48)], ids=str)
def test_float_inputs_with_a_scale(cuda, dtype, n, p, c, groups, pitch):
    g = torch.Generator(device="cuda").manual_seed(66)
    wide = (torch.randn(n, p, pitch, generator=g, device="cuda") + 1).to(dtype)
    x = wide[..., :c]
    scale = (torch.rand(c + 1, generator=g, device="cuda") * 4 - 2)[1:]   # 4-byte aligned, signed
    scale[c // 2] = 0
    _check(x, groups, scale)
    before = x.clone()
    ws = torch.empty(m.group_norm_workspace_bytes(x, groups, x), dtype=torch.uint8, device="cuda")
    want = m.group_norm(x.contiguous(), groups, scale=scale, activation="gelu")
    m.launch_group_norm(x, groups, x, scale=scale, activation="gelu", workspace=ws,
                        workspace_bytes=ws.numel())
    if pitch == c:
        assert torch.equal(x, want)
    assert bool(torch.isfinite(x.float()).all()) and not torch.equal(x, before)


def test_not_finite_values_under_a_scale_stay_in_their_groups(cuda):
    x = torch.randn(3, 500, 32, generator=torch.Generator(device="cuda").manual_seed(67), device="cuda")
    scale = torch.rand(32, device="cuda") + 0.5
    x[0, 0, 9], x[1, 499, 17], x[2, 250, 25] = float("nan"), float("inf"), -float("inf")
    y = m.group_norm(x, 4, scale=scale)
    for image, group in ((0, 1), (1, 2), (2, 3)):
        bad = torch.isnan(y[image]).view(500, 4, 8).all(2).all(0)
        assert bad.tolist() == [g == group for g in range(4)]
        assert int(torch.isnan(y[image]).sum()) == 500 * 8
