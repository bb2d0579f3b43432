"""The compiled binding shares the process's C++ runtime: a copy of its own would crash at the first error message."""
import subprocess

import pytest


@pytest.fixture(scope="module")
def native():
    import __graft_entry__
    __graft_entry__.build()
    from momoe._lib import native
    return native


def test_one_cpp_runtime(native):
    needed = subprocess.run(["readelf", "-d", native.__file__], capture_output=True, text=True).stdout
    assert "libstdc++.so.6" in needed


def test_errors_are_python_errors(native):
    import torch
    with pytest.raises(RuntimeError, match="cannot load"):
        native.bind("/nowhere/libmomoe_b200.so")
    for _ in range(3):
        with pytest.raises(RuntimeError, match="no CPU path"):
            native.rms_norm(torch.zeros(2, 8), torch.ones(8), None, 1e-6)
    with pytest.raises(TypeError):
        native.rms_norm(1, 2, 3, 4)
    assert native.launches() >= 0
