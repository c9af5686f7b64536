"""The native host calls of int8 products and the per-head norm and the Python path behind them: the same bits for
the calls both take, the Python path's results for all others."""

from __future__ import annotations

import gc

import pytest
import torch

from test_gpu_native_calls import both  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_products(both):  # noqa: F811
    from ltx_amd.kernels import gemm

    g = torch.Generator(device=DEV).manual_seed(0)
    for m, k, n in ((1, 128, 8), (3, 1024, 72), (68, 2048, 264), (300, 512, 1032), (40, 8192, 264)):
        w = gemm.make_weight(torch.randn(n, k, generator=g, device=DEV).bfloat16(),
                             torch.randn(n, generator=g, device=DEV), kind="int8")
        rows = gemm.quantize_rows_int8(torch.randn(m, k, generator=g, device=DEV))
        wide = torch.zeros(m, k + 16, dtype=torch.int8, device=DEV)
        wide[:, :k] = rows.codes
        res = torch.randn(m, n, generator=g, device=DEV).bfloat16()
        gate = torch.randn(n, generator=g, device=DEV)
        for x in (rows, gemm.Int8Rows(wide[:, :k], rows.scales)):
            for qlinear in (False, True):
                wt = gemm.LinearWeight("int8", w.w, w.scale, w.bias, qlinear=qlinear)
                both(lambda: gemm.linear(x, wt))
                both(lambda: gemm.linear(x, wt, sigmoid_from=n - 5))
                both(lambda: gemm.linear(x, wt, sigmoid_from=-3))
                both(lambda: gemm.linear(x, wt, epilogue=gemm.EPI_GELU))
                for epi in (gemm.EPI_RESIDUAL, gemm.EPI_RESIDUAL_ROUND):
                    both(lambda: gemm.linear(x, wt, epilogue=epi, residual=res, gate=gate))
                    both(lambda: gemm.linear(x, wt, epilogue=epi, residual=res[None], gate=gate[None]))
            both(lambda: gemm.linear(x, gemm.LinearWeight("int8", w.w, w.scale)))


def test_rows(both):  # noqa: F811
    from ltx_amd.kernels import gemm

    def pair(r):
        return r.codes, r.scales

    for rows, k in ((1, 16), (5, 160), (130, 1024)):
        for dtype in (torch.bfloat16, torch.float16, torch.float32):
            x = torch.randn(rows, k + 16, device=DEV).to(dtype)[:, :k]
            both(lambda: pair(gemm.quantize_rows_int8(x)))
            q = gemm.quantize_rows_int8(x)
            both(lambda: gemm.dequantize_rows_int8(q))
            both(lambda: pair(gemm.quantize_rows_int8(x.view(1, *x.shape))))


def test_headnorm(both):  # noqa: F811
    from ltx_amd.kernels import rope_ops

    f, b = rope_ops.headnorm_rotary, rope_ops.headnorm_rotary_grad
    inv, _ = rope_ops.rotary_frequencies(32)
    for shape, kv in (((1, 4, 64), 2), ((2, 9, 4, 64), 1), ((33, 3, 80), 3)):
        for dtype in (torch.bfloat16, torch.float32):
            q, gq = (torch.randn(shape, device=DEV).to(dtype) for _ in range(2))
            k, gk = (torch.randn(*shape[:-2], kv, shape[-1], device=DEV).to(dtype) for _ in range(2))
            w, v = (torch.randn(shape[-1], device=DEV) for _ in range(2))
            pos = torch.arange(shape[-3], device=DEV)
            for kw in (dict(), dict(layout="interleaved", eps=1e-3, weight_offset=1, factor=2)):
                for a, c in ((w, v), (None, v), (None, None)):
                    both(lambda: f(q, k, a, c, pos, inv, **kw))
                    both(lambda: b(gq, gk, q, k, a, c, pos, inv, **kw))
                both(lambda: f(q, None, w, None, pos, inv, **kw))
                both(lambda: b(gq, None, q, None, w, None, pos, inv, **kw))
                both(lambda: f(q, k, w, v, None, None, eps=1e-5))
                both(lambda: f(q, k, w, v, pos, inv, out=(torch.empty_like(q), None), **kw))
                both(lambda: b(gq, gk, q, k, w, v, pos, inv, out=(None, gk.clone()), **kw))


def test_outputs_are_ordinary_tensors():
    """What the native calls return: of the caller's device and allocator, inference tensors in inference mode only, and
    no part of a graph for inputs that record one."""
    from ltx_amd.kernels import gemm, rope_ops

    x = torch.randn(5, 64, device="cuda")
    q, pos = torch.randn(5, 2, 64, device="cuda", requires_grad=True), torch.arange(5, device="cuda")
    inv, _ = rope_ops.rotary_frequencies(64)
    rows = gemm.quantize_rows_int8(x)
    with torch.inference_mode():
        again = gemm.quantize_rows_int8(x)
    assert not rows.codes.is_inference() and again.codes.is_inference() and torch.equal(rows.codes, again.codes)
    y, _ = rope_ops.headnorm_rotary(q, None, None, None, pos, inv)
    assert not y.requires_grad and y.device == x.device
    gc.collect()  # (what earlier tests left)
    before = torch.cuda.memory_allocated()
    big = gemm.dequantize_rows_int8(gemm.quantize_rows_int8(torch.zeros(1024, 1024, device="cuda", dtype=torch.bfloat16)))
    assert torch.cuda.memory_allocated() - before >= big.numel() * 2
    assert big.untyped_storage().device == x.untyped_storage().device
    del big
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before
    for t in (rows.codes, rows.scales, y):  # as torch's own: resized, copied, added to
        t.resize_(4 * t.numel())
        t.clone().add_(1)
