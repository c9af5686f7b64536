"""Where the native host calls are loaded from, and what happens without them."""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

PACKAGE = Path(__file__).resolve().parents[1] / "ltx-2-mlx_amd"


@pytest.fixture
def built():
    from ltx_amd import _lib

    if not _lib.LIB_PATH.with_name("_calls.so").exists():
        pytest.skip("the library and its native calls are not built")
    return _lib


def _calls_file(folder: Path) -> str:
    """The file of ltx_amd._lib.CALLS (or None) in a process whose library is in ``folder``."""
    script = ("from ltx_amd import _lib; assert _lib.lib().ltx_version() > 0; "
              "print(_lib.CALLS and _lib.CALLS.__file__)")
    env = dict(os.environ, LTX_HIP_LIB=str(folder / "libltx_hip.so"), PYTHONPATH=str(PACKAGE))
    done = subprocess.run([sys.executable, "-c", script], env=env, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr
    return done.stdout.strip().splitlines()[-1]


def test_the_calls_beside_the_library_are_the_ones_loaded(built, tmp_path):
    os.symlink(built.LIB_PATH, tmp_path / "libltx_hip.so")
    assert _calls_file(tmp_path) == "None"
    shutil.copy(built.LIB_PATH.with_name("_calls.so"), tmp_path / "_calls.so")
    assert _calls_file(tmp_path) == str(tmp_path / "_calls.so")


def test_calls_that_do_not_load_leave_the_library_working(built, tmp_path):
    os.symlink(built.LIB_PATH, tmp_path / "libltx_hip.so")
    (tmp_path / "_calls.so").write_bytes(b"not a module")
    assert _calls_file(tmp_path) == "None"


def test_calls_built_for_another_torch_are_not_used(built, monkeypatch):
    handle = built.lib()
    path = built.LIB_PATH.with_name("_calls.so")
    assert built._load_calls(path, handle) is not None
    monkeypatch.setattr(built.torch, "__version__", "1.0")
    with pytest.warns(RuntimeWarning, match="built for"):
        assert built._load_calls(path, handle) is None
