"""Loading the compiled calls: only those built for the torch and Python that run,
and without them the operators go on through the checks in Python."""
import importlib.util
import subprocess
import sys
import warnings
from pathlib import Path

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


def _commands(*variables):
    """What make would run for everything, from the start."""
    csrc = Path(m.__file__).parent / "csrc"
    return subprocess.run(["make", "-n", "-B", "-C", str(csrc), f"PYTHON={sys.executable}", *variables],
                          capture_output=True, text=True, check=True).stdout


def test_library_builds_without_a_torch_that_has_cuda(tmp_path):
    torch_dir = Path(importlib.util.find_spec("torch").submodule_search_locations[0])
    assert ("torch_calls.so" in _commands()) == (torch_dir / "lib" / "libc10_cuda.so").exists()
    # A CPU build of torch: libc10, its headers, no libc10_cuda.
    (tmp_path / "lib").mkdir()
    (tmp_path / "lib" / "libc10.so").touch()
    (tmp_path / "include" / "c10" / "cuda").mkdir(parents=True)
    (tmp_path / "include" / "c10" / "cuda" / "CUDAStream.h").touch()
    for where in (tmp_path, tmp_path / "none", ""):
        out = _commands(f"TORCH={where}")
        assert "libint8conv.so" in out and "torch_calls.cpp" not in out
