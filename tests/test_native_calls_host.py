"""The native host calls against stand-ins for the entry points, on host
tensors: what they pass on, what they raise, and that nothing is launched twice."""

from __future__ import annotations

import ctypes
import importlib.util
import shutil

import pytest
import torch

OK, INVALID, UNSUPPORTED, HIP, ALIGN = 0, -1, -2, -3, -4
HOST = (-1, 0)  # device and stream of host tensors


@pytest.fixture
def calls(tmp_path, monkeypatch):
    """A copy of the module whose entry points return ``calls.status`` and count,
    taking the place of the library's (ltx_amd._lib.CALLS)."""
    from ltx_amd import _lib

    if not _lib.LIB_PATH.with_name("_calls.so").exists():
        pytest.skip("_calls.so not built")
    _lib.lib()
    copy = tmp_path / "_calls.so"
    shutil.copy(_lib.LIB_PATH.with_name("_calls.so"), copy)
    spec = importlib.util.spec_from_file_location("stand_in._calls", copy)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)

    class Calls:
        status = OK
        count = 0
        native = module

    state, keep = Calls(), []
    for name in _lib._CALLS_ENTRIES:
        size = name in _lib.SIZES

        def stub(*_, size=size):
            if size:
                return 0
            state.count += 1
            return state.status

        keep.append(ctypes.CFUNCTYPE(ctypes.c_int64 if size else ctypes.c_int, *_lib.SIGNATURES[name])(stub))
    module.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in keep))
    state.keep = keep
    monkeypatch.setattr(_lib, "CALLS", module)
    monkeypatch.setattr(_lib, "fast_stream", lambda t: HOST)
    monkeypatch.setattr(_lib, "launch", lambda *a: pytest.fail("the call was made again"))
    return state


def _every_call():
    from ltx_amd.kernels import gemm, rope_ops

    w = gemm.LinearWeight("mxfp4", torch.zeros(64, 64, dtype=torch.uint8), torch.zeros(1, 64, dtype=torch.int32))
    rows = gemm.Mx4Rows(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(1, 4, dtype=torch.int32))
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    res, gate = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(64)
    q, k, pos = torch.zeros(4, 2, 64), torch.zeros(4, 1, 64), torch.arange(4)
    inv, _ = rope_ops.rotary_frequencies(64, device="cpu")
    add = dict(epilogue=gemm.EPI_RESIDUAL, residual=res, gate=gate, out=res)
    return [lambda: gemm.linear(x, w), lambda: gemm.linear(x, w, **add), lambda: gemm.linear(rows, w, **add),
            lambda: gemm.quantize_rows_mxfp4(x), lambda: gemm.dequantize_rows_mxfp4(rows),
            lambda: rope_ops.rotary(q, k, pos, inv), lambda: rope_ops.rotary(q, k, pos, inv, out=(q, k)),
            lambda: rope_ops.rotary(q, None, pos, inv)]


def test_a_failed_launch_raises_and_is_not_made_again(calls):
    from ltx_amd import _lib

    for status in (HIP, -5, 7):
        for i, call in enumerate(_every_call()):
            calls.status, calls.count = status, 0
            with pytest.raises(_lib.LtxKernelError):
                call()
            assert calls.count == 1, (i, status)


def test_a_launch_is_made_once(calls):
    for i, call in enumerate(_every_call()):
        calls.count = 0
        assert call() is not None
        assert calls.count == 1, i


def test_a_refusal_goes_to_the_python_path(calls):
    for status in (INVALID, UNSUPPORTED, ALIGN):
        for call in _every_call():
            calls.status = status
            with pytest.raises(ValueError, match="on one GPU"):  # its checks, met by host tensors
                call()


@pytest.mark.parametrize("rows,k", [(5, 128), (3, 256), (70, 640)])
def test_scale_words_are_read_up_to_a_multiple_of_four_rows(calls, monkeypatch, rows, k):
    """Words whose memory ends with the rows go to the kernel as a copy that goes on;
    a column range of wider words goes as it is, natively."""
    from ltx_amd import _lib
    from ltx_amd.kernels import gemm

    seen = []
    monkeypatch.setattr(_lib, "same_device", lambda *t: -1)
    monkeypatch.setattr(_lib, "launch", lambda *a: seen.append(a) or 0)
    w = gemm.LinearWeight("mxfp4", torch.zeros(64, k // 2, dtype=torch.uint8),
                          torch.zeros(k // 128, 64, dtype=torch.int32))
    codes = torch.zeros(rows, k // 2, dtype=torch.uint8)
    ld, words = -(-rows // 4) * 4, k // 128
    wide = torch.arange(words * (ld + 8), dtype=torch.int32).view(words, ld + 8)
    held = []
    pad = torch.nn.functional.pad
    monkeypatch.setattr(torch.nn.functional, "pad", lambda *a, **kw: held.append(pad(*a, **kw)) or held[-1])
    for given, whole in ((wide[:, 8:], True), (wide[:, 4:4 + rows], True),
                         (wide.flatten()[8:8 + (words - 1) * (ld + 8) + rows].clone().as_strided(
                             (words, rows), (ld + 8, 1)), False)):
        calls.count, seen[:], held[:] = 0, [], []
        gemm.linear(gemm.Mx4Rows(codes, given), w)
        assert calls.count == int(whole) and len(seen) == int(not whole)
        if not whole:
            _, name, _, _, ptr, stride = seen[0][:6]
            assert name == "ltx_gemm_mx4_bf16" and ptr == held[0].data_ptr() and stride == ld
            assert held[0].shape == (words, ld) and torch.equal(held[0][:, :rows], given)


@pytest.mark.parametrize("native", [True, False])
def test_outputs_over_other_operands_are_refused(calls, monkeypatch, native):
    """A given output that shares memory with anything that a product reads."""
    from ltx_amd import _lib
    from ltx_amd.kernels import gemm

    if not native:
        monkeypatch.setattr(_lib, "CALLS", None)
    buf = torch.zeros(1 << 15, dtype=torch.uint8)

    def at(offset, dtype, *shape):
        return buf[offset:].view(dtype)[:torch.Size(shape).numel()].view(shape)

    free = dict(x=torch.zeros(4, 128, dtype=torch.bfloat16), xc=torch.zeros(4, 64, dtype=torch.uint8),
                xs=torch.zeros(1, 4, dtype=torch.int32), w=torch.zeros(64, 64, dtype=torch.uint8),
                ws=torch.zeros(1, 64, dtype=torch.int32), bias=torch.zeros(64), gate=torch.zeros(64),
                res=torch.zeros(4, 64, dtype=torch.bfloat16))
    out = at(4096, torch.bfloat16, 4, 64)  # bytes 4096 to 4608
    over = dict(x=at(4608 - 16, torch.bfloat16, 4, 128), xc=at(4096 - 240, torch.uint8, 4, 64),
                xs=at(4096, torch.int32, 1, 4), w=at(4352, torch.uint8, 64, 64), ws=at(4096 - 64, torch.int32, 1, 64),
                bias=at(4600, torch.float32, 64), gate=at(4096 - 252, torch.float32, 64),
                res=at(4096 - 16, torch.bfloat16, 4, 64))

    def product(t, quantised):
        x = gemm.Mx4Rows(t["xc"], t["xs"]) if quantised else t["x"]
        return gemm.linear(x, gemm.LinearWeight("mxfp4", t["w"], t["ws"], t["bias"]), epilogue=gemm.EPI_RESIDUAL,
                           residual=t["res"], gate=t["gate"], out=out)

    for quantised in (False, True):
        for name in free:
            if name in (("x",) if quantised else ("xc", "xs")):
                continue
            with pytest.raises(ValueError, match="overlaps"):
                product({**free, name: over[name]}, quantised)
        assert calls.count == 0
        if native:
            assert product(free, quantised) is out and calls.count == 1
            assert product({**free, "res": out}, quantised) is out and calls.count == 2  # in place
            calls.count = 0


@pytest.mark.parametrize("native", [True, False])
def test_bias_and_gate_of_many_axes(calls, monkeypatch, native):
    """N values in any shape; the overlap check counts their bytes, not their axes."""
    from ltx_amd import _lib
    from ltx_amd.kernels import gemm

    if not native:
        monkeypatch.setattr(_lib, "CALLS", None)
    shape = (1, 2, 2, 2, 2, 2, 2)
    w = torch.zeros(64, 64, dtype=torch.uint8), torch.zeros(1, 64, dtype=torch.int32)
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    buf = torch.zeros(1024, dtype=torch.float32)  # out in bytes 0 to 512, the values after it or over its end
    out = buf[:128].view(torch.bfloat16).view(4, 64)
    apart, over = buf[128:192].view(shape), buf[127:191].view(shape)
    for bias, gate, fine in ((apart, apart, True), (over, apart, False), (apart, over, False)):
        def product():
            return gemm.linear(x, gemm.LinearWeight("mxfp4", *w, bias), epilogue=gemm.EPI_RESIDUAL, residual=out,
                               gate=gate, out=out)

        calls.count = 0
        if not fine:
            with pytest.raises(ValueError, match="overlaps"):
                product()
        elif native:
            assert product() is out and calls.count == 1
        else:
            with pytest.raises(ValueError, match="on one GPU"):
                product()
