"""What is built for whom: the C library alone, and the module that Python calls go through where it can be had."""
import os
import subprocess
import sys

import pytest
import torch

from tests.test_dense_block_cpu import _adapters, _append, _paged
from wsvd_b200 import _lib, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def no_module(monkeypatch, tmp_path):
    """As on a machine without a C++ compiler, in a process that has not called an operator yet."""
    monkeypatch.setattr(_lib, "bind_path", lambda: str(tmp_path / "_bind.so"))
    monkeypatch.setattr(_lib, "_bind", None)
    monkeypatch.setattr(ops, "_fast", None)
    monkeypatch.setenv("CXX", "/bin/false")
    return tmp_path


def test_without_the_module_calls_take_the_long_way(no_module):
    with pytest.warns(RuntimeWarning, match="ctypes"):
        with pytest.raises(ValueError, match="must be a CUDA tensor"):
            _adapters()()
    for call in (_append(), _paged(), _adapters(out=torch.zeros(3, 24, dtype=torch.float16))):  # (said once)
        with pytest.raises(ValueError, match="must be a CUDA tensor"):
            call()
    assert os.listdir(no_module) == ["_bind.so.lock"]


def test_the_library_does_not_wait_for_the_module(no_module, monkeypatch):
    monkeypatch.setattr(_lib, "_lib", None)
    assert _lib.lib().wsvd_abi_version() == 1
    assert not os.listdir(no_module)


def test_build_says_that_the_module_is_missing(no_module):
    with pytest.warns(RuntimeWarning, match="bind.cpp was not built"):
        assert _lib.build() == _lib.LIB_PATH


def test_the_module_is_one_pythons_and_one_torchs():
    name = os.path.basename(_lib.bind_path())
    assert sys.implementation.cache_tag in name and torch.__version__ in name


def test_the_library_loads_where_there_is_no_torch():
    """In a process that cannot import torch, as a user of the C entries through ctypes may have it."""
    code = ("import importlib.util, sys\n"
            "sys.modules['torch'] = None\n"
            f"spec = importlib.util.spec_from_file_location('lib_alone', {os.path.join(ROOT, 'wsvd_b200', '_lib.py')!r})\n"
            "m = importlib.util.module_from_spec(spec)\n"
            "spec.loader.exec_module(m)\n"
            "assert m.lib().wsvd_abi_version() == 1\n"
            "try:\n"
            "    m.bind()\n"
            "except m.NO_BIND:\n"
            "    print('no module')\n")
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert res.returncode == 0 and res.stdout == "no module\n", res.stderr
