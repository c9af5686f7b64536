"""Building the native host calls: a machine without what they need still builds the library."""

from __future__ import annotations

import shutil
import sysconfig

import pytest


@pytest.fixture
def build_lib(tmp_path, monkeypatch):
    import build_lib

    monkeypatch.setattr(build_lib, "LIB_PATH", tmp_path / "libltx_hip.so")
    return build_lib


def _none_is_left(build_lib, capsys, named: str):
    stale = build_lib.LIB_PATH.with_name("_calls.so")
    stale.write_bytes(b"an earlier build")
    assert build_lib.build_calls() is None
    assert not stale.exists() and named in capsys.readouterr().out


def test_without_a_host_compiler(build_lib, monkeypatch, capsys):
    monkeypatch.setattr(shutil, "which", lambda name, *a, **kw: None)
    _none_is_left(build_lib, capsys, "compiler")


def test_without_python_headers(build_lib, monkeypatch, tmp_path, capsys):
    monkeypatch.setattr(sysconfig, "get_paths", lambda *a, **kw: {"include": str(tmp_path)})
    _none_is_left(build_lib, capsys, "Python.h")


def test_without_torch_headers(build_lib, monkeypatch, capsys):
    from torch.utils import cpp_extension

    monkeypatch.setattr(cpp_extension, "include_paths", lambda *a, **kw: [])
    _none_is_left(build_lib, capsys, "python_variable.h")
