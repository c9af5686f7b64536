"""What the native host calls allocate is seen by whoever looks at torch's own allocations: a dispatch mode, and the
fill of uninitialised memory."""

from __future__ import annotations

import ctypes
import importlib.util
import shutil

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

pytestmark = pytest.mark.gpu
DEV = "cuda"


class _Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.sizes = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if "empty" in str(func):
            self.sizes.append(tuple(out.shape))
        return out


def _every_call():
    """(call, the shapes of what it returns)."""
    from ltx_amd.kernels import gemm, rope_ops

    x = torch.randn(5, 256, device=DEV).bfloat16()
    w = torch.randn(64, 256, device=DEV).bfloat16()
    w4, w8 = gemm.make_weight(w, kind="mxfp4"), gemm.make_weight(w, kind="int8")
    x4, x8 = gemm.quantize_rows_mxfp4(x), gemm.quantize_rows_int8(x)
    q, k = torch.randn(5, 2, 64, device=DEV), torch.randn(5, 1, 64, device=DEV)
    pos, nw = torch.arange(5, device=DEV), torch.randn(64, device=DEV)
    inv, _ = rope_ops.rotary_frequencies(64)
    heads = [(5, 2, 64), (5, 1, 64)]
    return [(lambda: gemm.quantize_rows_mxfp4(x), [(5, 128), (2, 8)]), (lambda: gemm.dequantize_rows_mxfp4(x4), [(5, 256)]),
            (lambda: gemm.linear(x, w4), [(5, 64)]), (lambda: gemm.linear(x4, w4), [(5, 64)]),
            (lambda: gemm.quantize_rows_int8(x), [(5, 256), (5,)]), (lambda: gemm.dequantize_rows_int8(x8), [(5, 256)]),
            (lambda: gemm.linear(x8, w8), [(5, 64)]), (lambda: rope_ops.rotary(q, k, pos, inv), heads),
            (lambda: rope_ops.headnorm_rotary(q, k, nw, nw, pos, inv), heads),
            (lambda: rope_ops.headnorm_rotary_grad(q, k, q, k, nw, nw, pos, inv), heads + [(64,), (64,)])]


def test_a_dispatch_mode_sees_every_output():
    for i, (call, shapes) in enumerate(_every_call()):
        call()
        with _Seen() as seen:
            call()
        left = list(seen.sizes)
        for shape in shapes:
            assert shape in left, (i, shape, seen.sizes)
            left.remove(shape)
    torch.cuda.synchronize()


def test_uninitialised_memory_is_filled():
    """The scale words past the rows of an MXFP4 operand are not written: with torch's fill they hold its value."""
    from ltx_amd.kernels import gemm

    x = torch.randn(5, 256, device=DEV).bfloat16()
    for _ in range(3):  # memory that the allocator gives out again
        torch.zeros(2, 8, dtype=torch.int32, device=DEV)
    torch.use_deterministic_algorithms(True)
    before = torch.utils.deterministic.fill_uninitialized_memory
    torch.utils.deterministic.fill_uninitialized_memory = True
    try:
        words = gemm.quantize_rows_mxfp4(x).scales
    finally:
        torch.use_deterministic_algorithms(False)
        torch.utils.deterministic.fill_uninitialized_memory = before
    assert (words[:, 5:] == torch.iinfo(torch.int32).max).all(), words


def test_a_first_call_under_a_mode_settles_nothing(tmp_path):
    """A freshly loaded module whose first call meets a mode that answers allocations itself."""
    from ltx_amd import _lib

    _lib.lib()
    copy = tmp_path / "_calls.so"
    shutil.copy(_lib.LIB_PATH.with_name("_calls.so"), copy)
    spec = importlib.util.spec_from_file_location("fresh._calls", copy)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)

    class Elsewhere(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **{**(kwargs or {}), "device": "cpu"} if "empty" in str(func) else kwargs or {})

    def address(f):
        return ctypes.cast(f, ctypes.c_void_p).value

    x = torch.randn(5, 256, device=DEV).bfloat16()
    where = _lib.fast_stream(x)
    refuse = [ctypes.CFUNCTYPE(ctypes.c_int64 if n in _lib.SIZES else ctypes.c_int, *_lib.SIGNATURES[n])(lambda *_: -1)
              for n in _lib._CALLS_ENTRIES]  # stand-ins that launch nothing
    module.bind(*map(address, refuse))
    with Elsewhere():
        assert module.quantize8(x, *where) is None
    module.bind(*(address(getattr(_lib.lib(), n)) for n in _lib._CALLS_ENTRIES))
    codes, scales = module.quantize8(x, *where)
    assert codes.device == x.device and scales.device == x.device
    assert codes.untyped_storage().device == x.device
