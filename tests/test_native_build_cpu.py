"""A binding that was compiled for another torch or Python is rebuilt, and not loaded."""
import importlib.util
import os
import shutil
import types

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def build():
    import __graft_entry__
    __graft_entry__.build()
    spec = importlib.util.spec_from_file_location("momoe_build", os.path.join(ROOT, "momoe-impl_b200", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_binding_of_other_versions_is_stale(build, tmp_path, monkeypatch):
    copy = str(tmp_path / "_native.so")
    shutil.copy(build.BINDING_PATH, copy)
    assert not build.binding_stale() and not build.binding_stale(copy)
    assert build.binding_stale(str(tmp_path / "missing.so"))
    import torch
    monkeypatch.setattr(torch, "__version__", torch.__version__ + "0")
    assert build.binding_stale(copy)


def test_binding_of_other_versions_is_not_loaded(build):
    from momoe import _lib
    _lib.require_fitting(_lib.native)
    for other in (types.SimpleNamespace(built_for="torch 1.0, Python 3.8"), types.SimpleNamespace()):
        with pytest.raises(ImportError, match="build.py"):
            _lib.require_fitting(other)
