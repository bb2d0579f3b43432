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


def test_package_without_the_binding(build, tmp_path):
    """The layer in 16 bits does not need it; the operators that do name the build command."""
    import subprocess
    import sys
    home = tmp_path / "momoe"
    shutil.copytree(os.path.dirname(build.LIB_PATH), home, ignore=shutil.ignore_patterns("*.so", "__pycache__"))
    os.symlink(build.LIB_PATH, home / "libmomoe_b200.so")
    code = """
import torch, momoe, momoe.norm, momoe.balance, momoe.fp8
from momoe import _lib, ops
assert ops.launch_count() == 0
for use in (lambda: momoe.norm.rms_norm(torch.zeros(2, 8), torch.ones(8)), lambda: _lib.native.bind):
    for _ in range(2):
        try:
            use()
        except ImportError as e:
            assert "build.py" in str(e), e
        else:
            raise AssertionError
"""
    got = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, PYTHONPATH=str(tmp_path)), capture_output=True, text=True)
    assert got.returncode == 0, got.stderr
    shutil.copy(build.BINDING_PATH, home / "_native.so")
    code = """
import torch, momoe.norm
from momoe import _lib, ops
assert ops.launch_count() == 0
try:
    momoe.norm.rms_norm(torch.zeros(2, 8), torch.ones(8))
except RuntimeError as e:
    assert "no CPU path" in str(e), e
assert ops.launch_count() == 0 and "launches" in vars(_lib.native) and _lib.native.__file__.endswith("_native.so")
"""
    got = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, PYTHONPATH=str(tmp_path)), capture_output=True, text=True)
    assert got.returncode == 0, got.stderr
