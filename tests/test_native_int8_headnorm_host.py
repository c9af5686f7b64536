"""The native host calls of int8 products and the per-head norm against stand-ins for the entry points, on host
tensors: a launch is made once, a failed one raises, refusals and overlaps go to the Python path's errors."""

from __future__ import annotations

import pytest
import torch

from test_native_calls_host import ALIGN, HIP, INVALID, UNSUPPORTED, calls  # noqa: F401


def _operands():
    from ltx_amd.kernels import gemm, rope_ops

    rows = gemm.Int8Rows(torch.zeros(4, 128, dtype=torch.int8), torch.zeros(4))
    w = gemm.LinearWeight("int8", torch.zeros(64, 128, dtype=torch.int8), torch.zeros(64), torch.zeros(64))
    q, k, pos = torch.zeros(4, 2, 64), torch.zeros(4, 1, 64), torch.arange(4)
    inv, _ = rope_ops.rotary_frequencies(64, device="cpu")
    return rows, w, q, k, pos, inv


def _every_call():
    from ltx_amd.kernels import gemm, rope_ops

    rows, w, q, k, pos, inv = _operands()
    res, gate, nw = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(64), torch.zeros(64)
    add = dict(epilogue=gemm.EPI_RESIDUAL, residual=res, gate=gate, out=res)
    f, b = rope_ops.headnorm_rotary, rope_ops.headnorm_rotary_grad
    gq, gk = q.clone(), k.clone()
    return [lambda: gemm.quantize_rows_int8(torch.zeros(4, 64)), lambda: gemm.dequantize_rows_int8(rows),
            lambda: gemm.linear(rows, w), lambda: gemm.linear(rows, w, **add), lambda: gemm.linear(rows, w, sigmoid_from=3),
            lambda: f(q, k, nw, nw, pos, inv), lambda: f(q, k, nw, nw, pos, inv, out=(q, k)),
            lambda: f(q, None, None, None, pos, inv), lambda: f(q[None], k[None], None, nw, pos[None], inv),
            lambda: b(gq, gk, q, k, nw, nw, pos, inv), lambda: b(gq, gk, q, k, nw, None, pos, inv, out=(gq, k)),
            lambda: b(gq, None, q, None, None, None, pos, inv), lambda: b(gq, None, q, None, nw, None, pos, inv)]


def test_a_launch_is_made_once(calls):  # noqa: F811
    for i, call in enumerate(_every_call()):
        calls.count = 0
        assert call() is not None
        assert calls.count == 1, i


def test_a_failed_launch_raises_and_is_not_made_again(calls):  # noqa: F811
    from ltx_amd import _lib

    for status in (HIP, -5, 7):
        for i, call in enumerate(_every_call()):
            calls.status, calls.count = status, 0
            with pytest.raises(_lib.LtxKernelError):
                call()
            assert calls.count == 1, (i, status)


def test_a_refusal_goes_to_the_python_path(calls):  # noqa: F811
    for status in (INVALID, UNSUPPORTED, ALIGN):
        for call in _every_call():
            calls.status = status
            with pytest.raises(ValueError, match="on one GPU"):  # its checks, met by host tensors
                call()


def test_results_have_their_places(calls):  # noqa: F811
    from ltx_amd.kernels import rope_ops

    _, _, q, k, pos, inv = _operands()
    w = torch.zeros(64)
    a, b = rope_ops.headnorm_rotary(q, None, w, None, pos, inv)
    assert a.shape == q.shape and b is None
    got = rope_ops.headnorm_rotary_grad(q, k, q, k, None, w, pos, inv)
    assert [None if t is None else t.shape for t in got] == [q.shape, k.shape, None, w.shape]
    got = rope_ops.headnorm_rotary_grad(q, k, q, k, None, None, pos, inv)
    assert got[2] is None and got[3] is None


@pytest.mark.parametrize("native", [True, False])
def test_outputs_over_other_operands_are_refused(calls, monkeypatch, native):  # noqa: F811
    from ltx_amd import _lib
    from ltx_amd.kernels import gemm, rope_ops

    if not native:
        monkeypatch.setattr(_lib, "CALLS", None)
    buf = torch.zeros(1 << 15, dtype=torch.uint8)

    def at(offset, dtype, *shape):
        return buf[offset:].view(dtype)[:torch.Size(shape).numel()].view(shape)

    free = dict(x=torch.zeros(4, 128, dtype=torch.int8), xs=torch.zeros(4), w=torch.zeros(64, 128, dtype=torch.int8),
                ws=torch.zeros(64), bias=torch.zeros(64), gate=torch.zeros(64),
                res=torch.zeros(4, 64, dtype=torch.bfloat16))
    out = at(4096, torch.bfloat16, 4, 64)  # bytes 4096 to 4608
    over = dict(x=at(4608 - 16, torch.int8, 4, 128), xs=at(4600, torch.float32, 4), w=at(4352, torch.int8, 64, 128),
                ws=at(4096 - 252, torch.float32, 64), bias=at(4604, torch.float32, 64),
                gate=at(4096, torch.float32, 64), res=at(4096 - 16, torch.bfloat16, 4, 64))

    def product(t):
        return gemm.linear(gemm.Int8Rows(t["x"], t["xs"]), gemm.LinearWeight("int8", t["w"], t["ws"], t["bias"]),
                           epilogue=gemm.EPI_RESIDUAL, residual=t["res"], gate=t["gate"], out=out)

    for name in free:
        with pytest.raises(ValueError, match="overlaps"):
            product({**free, name: over[name]})
    assert calls.count == 0
    if native:
        assert product(free) is out and product({**free, "res": out}) is out and calls.count == 2

    calls.count = 0
    oq, ok = at(8192, torch.float32, 4, 2, 64), at(8192 + 2048, torch.float32, 4, 1, 64)
    heads = dict(gq=torch.zeros(4, 2, 64), gk=torch.zeros(4, 1, 64), q=torch.zeros(4, 2, 64), k=torch.zeros(4, 1, 64),
                 wq=torch.zeros(64), wk=torch.zeros(64), pos=torch.arange(4), inv=torch.zeros(32, dtype=torch.float64))
    last = 8192 + 2048 + 1024
    over = dict(gq=at(8192 - 4, torch.float32, 4, 2, 64), gk=at(last - 4, torch.float32, 4, 1, 64),
                q=at(8192 + 4, torch.float32, 4, 2, 64), k=at(8192, torch.float32, 4, 1, 64),
                wq=at(8192 + 2000, torch.float32, 64), wk=at(last - 4, torch.float32, 64),
                pos=at(8192, torch.int64, 4), inv=at(last - 8, torch.float64, 32))

    def grad(t, **kw):
        return rope_ops.headnorm_rotary_grad(t["gq"], t["gk"], t["q"], t["k"], t["wq"], t["wk"], t["pos"], t["inv"],
                                             out=(oq, ok), **kw)

    def forward(t):
        return rope_ops.headnorm_rotary(t["q"], t["k"], t["wq"], t["wk"], t["pos"], t["inv"], out=(oq, ok))

    for name in heads:
        with pytest.raises(ValueError, match="overlaps"):
            grad({**heads, name: over[name]})
        if name[0] != "g":
            with pytest.raises(ValueError, match="overlaps"):
                forward({**heads, name: over[name]})
    assert calls.count == 0
    if native:
        for own in (dict(q=oq), dict(gq=oq, gk=ok), dict(q=oq, gk=ok), dict(k=ok, q=oq)):
            assert grad({**heads, **own})[0] is oq
        assert forward({**heads, "q": oq, "k": ok})[1] is ok
        assert calls.count == 5
