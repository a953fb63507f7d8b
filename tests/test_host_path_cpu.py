"""CPU: the native host path is built by the test session, loads beside the library it was built with, and leaves every call on tensors that are not
on a GPU to the Python layer."""
import shutil

import pytest
import torch


@pytest.fixture
def native(built_lib):
    from flaggems_sglang_b200 import _build
    from flaggems_sglang_b200.ops import _host
    if shutil.which("g++") is None:
        pytest.skip("no compiler: the package does without the native host path")
    assert _build.build_fastcall() == _build.FASTCALL_PATH and _build.FASTCALL_PATH.exists()
    return _host.fast()


def test_it_is_built_and_loads(native):
    from flaggems_sglang_b200 import _lib
    assert native and native.version == _lib.VERSION and torch.__version__.startswith(native.torch_version)


def test_it_leaves_cpu_tensors(native):
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    q, s = torch.zeros(8, 128).to(torch.float8_e4m3fn), torch.ones(1, 1)
    status = torch.zeros(1, dtype=torch.int32)
    assert native.norm(False, True, False, False, False, 1.0, 1e-6, 0.0, x, None, None, None, None, None, None) is None
    assert native.activation(0, 1.0, 0.0, False, x) is None
    assert native.linear(x, q, s, None, None, status) is None
    assert native.norm() is None and native.activation() is None and native.linear() is None


def test_a_stale_one_is_built_again(native, tmp_path, monkeypatch):
    """Older than its sources: compiled anew.  No compiler: reported, and None."""
    from flaggems_sglang_b200 import _build
    target = tmp_path / "_fastcall.so"
    target.write_bytes(b"")
    import os
    os.utime(target, (1, 1))
    monkeypatch.setattr(_build, "FASTCALL_PATH", target)
    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        raise OSError("no compiler")

    monkeypatch.setattr(_build.subprocess, "run", run)
    assert _build.build_fastcall() is None and len(calls) == 1
    os.utime(target)
    assert _build.build_fastcall() == target and len(calls) == 1
