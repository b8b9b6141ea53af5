"""Loading the compiled calls: only those built for the torch and Python that run,
and without them the operators go on through the checks in Python."""
import sys
import warnings

import pytest
import torch

import int8_kernel_lab_b200 as m
from int8_kernel_lab_b200 import operators

HERE = f"torch {torch.__version__}, Python {sys.version_info[0]}.{sys.version_info[1]}"


@pytest.fixture
def fresh(monkeypatch):
    """operators as before its first call."""
    monkeypatch.setattr(operators, "_torch", None)
    monkeypatch.setattr(operators, "_calls", None)
    return monkeypatch


def test_built_calls_are_those_of_this_torch(fresh):
    if not operators._CALLS_PATH.exists():
        pytest.skip("torch_calls.so was not built")
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        operators._load_torch()
    assert operators._calls.built_for == HERE


@pytest.mark.parametrize("name,text", [
    ("torch_calls.so", "not a shared object"),
    ("torch_calls.py", "built_for = 'torch 1.0, Python 3.1'"),
    ("torch_calls.py", "raise ImportError('undefined symbol')"),
    ("torch_calls.py", "pass")])
def test_other_files_are_left_alone(fresh, tmp_path, name, text):
    path = tmp_path / name
    path.write_text(text)
    fresh.setattr(operators, "_CALLS_PATH", path)
    with pytest.warns(RuntimeWarning, match="built again"):
        operators._load_torch()
    assert operators._calls is None and operators._torch is torch
    with warnings.catch_warnings():
        warnings.simplefilter("error")      # once is enough
        with pytest.raises(ValueError):
            m.quantize_rows(torch.zeros(3))


def test_missing_file_is_not_worth_a_warning(fresh, tmp_path):
    fresh.setattr(operators, "_CALLS_PATH", tmp_path / "none.so")
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        operators._load_torch()
    assert operators._calls is None
