"""Arguments beyond the descriptors' fields are refused like other wrong ones."""
import pytest
import torch

import int8_kernel_lab_b200 as m
from test_operators_cpu import _Fake, device0  # noqa: F401

F32, I8 = torch.float32, torch.int8


@pytest.mark.parametrize("change", [
    dict(groups=1 << 40), dict(groups=-(1 << 40)),
    dict(x=_Fake(F32, (1, 1, (1 << 32) + 32)), y=_Fake(F32, (1, 1, (1 << 32) + 32)))])
def test_group_norm(device0, change):  # noqa: F811
    t = dict(x=_Fake(F32, (2, 9, 32)), groups=4, y=_Fake(F32, (2, 9, 32)))
    t.update(change)
    with pytest.raises(ValueError, match="range"):
        m.launch_group_norm(t.pop("x"), t.pop("groups"), t.pop("y"), **t)


@pytest.mark.parametrize("change", [
    dict(eps=1e300), dict(y=_Fake(I8, (2, 9, 32)), out_scale=1e300)])
def test_group_norm_in_fp32(device0, change):  # noqa: F811
    t = dict(x=_Fake(F32, (2, 9, 32)), y=_Fake(F32, (2, 9, 32)))
    t.update(change)
    with pytest.raises(m.Int8ConvError):
        m.launch_group_norm(t.pop("x"), 4, t.pop("y"), **t)
