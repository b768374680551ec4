"""What decides whether the libraries are built again, and what a call module of another torch or Python says."""
import sys
import sysconfig
from types import SimpleNamespace

import pytest
import torch

from saga_b200 import build as B


@pytest.fixture
def built():
    if not B.up_to_date():
        pytest.skip("the libraries were built from other sources")


@pytest.mark.parametrize("what", ["torch version", "C++ ABI of torch", "Python", "compiler"])
def test_the_call_module_is_built_again_for_another(what, built, monkeypatch):
    if what == "torch version":
        monkeypatch.setattr(torch, "__version__", "9.9.9")
    elif what == "C++ ABI of torch":
        monkeypatch.setattr(torch._C, "_GLIBCXX_USE_CXX11_ABI", not torch._C._GLIBCXX_USE_CXX11_ABI)
    elif what == "Python":
        monkeypatch.setattr(sys, "version", "4.0.0")
    else:
        monkeypatch.setenv("CXX", "another-g++")
    assert not B.up_to_date()


def test_the_library_needs_no_torch(built, monkeypatch):
    """Without torch the C-ABI library is built (and found up to date) by itself."""
    monkeypatch.setitem(sys.modules, "torch", None)
    assert B._fast_command("x.so") is None
    digest = B._digest()
    with open(B.STAMP) as f:
        assert f.read().split() != [digest]   # the library with its module is another build
    monkeypatch.setattr(B, "FAST", "/nonexistent")
    monkeypatch.setattr(B, "_stamped", lambda: digest)
    assert B.up_to_date()


def test_the_call_module_is_named_for_its_python():
    assert B.FAST.endswith("_fastcall" + sysconfig.get_config_var("EXT_SUFFIX"))


def test_a_call_module_of_another_torch_is_refused():
    from saga_b200 import kv4
    assert torch.__version__.startswith(kv4._fast.torch_version)
    kv4._check_built_for(kv4._fast)
    for module in (SimpleNamespace(torch_version="1.0.0"), SimpleNamespace()):
        with pytest.raises(ImportError, match="saga_b200.build"):
            kv4._check_built_for(module)
