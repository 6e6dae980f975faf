"""The binding of the paged operators is rebuilt for, and loaded with, the Python and torch it was compiled against."""
import os

import pytest

from zs_b200 import ZsError, build, paged


@pytest.fixture
def binding(tmp_path, monkeypatch):
    """A binding newer than its sources, compiled against what the stamp says."""
    so, abi = tmp_path / "_paged.so", tmp_path / "_paged.so.abi"
    so.write_bytes(b"")
    newest = max((build.CSRC / "zs_paged_py.cpp").stat().st_mtime, (build.INCLUDE / "zs.h").stat().st_mtime)
    os.utime(so, (newest + 10, newest + 10))
    monkeypatch.setattr(build, "BINDING", so)
    monkeypatch.setattr(build, "BINDING_ABI", abi)
    return abi


def test_another_torch_or_python_asks_for_a_build(binding, monkeypatch):
    import sysconfig

    import torch

    assert build.binding_needs_build()                       # no stamp: an unknown one
    binding.write_text(build.binding_abi())
    assert not build.binding_needs_build()
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", "9.9.9")
        assert build.binding_needs_build()
    with monkeypatch.context() as m:
        m.setattr(torch._C, "_GLIBCXX_USE_CXX11_ABI", not torch._C._GLIBCXX_USE_CXX11_ABI)
        assert build.binding_needs_build()
    with monkeypatch.context() as m:
        m.setattr(sysconfig, "get_config_var", lambda name: "cpython-399-other")
        assert build.binding_needs_build()
    assert not build.binding_needs_build()


def test_a_binding_for_another_torch_is_not_used(monkeypatch):
    if not (build.LIB.exists() and build.BINDING.exists()):
        pytest.skip("not built")
    monkeypatch.setattr(paged, "_BINDING", None)
    assert paged._binding().abi == build.binding_abi()
    for other in ("cpython-39 torch 1.0 cxx11abi 0", ""):
        monkeypatch.setattr(paged, "_BINDING", None)
        monkeypatch.setattr(paged, "binding_abi", lambda: other)
        with pytest.raises(ZsError, match="another Python or torch"):
            paged._binding()
