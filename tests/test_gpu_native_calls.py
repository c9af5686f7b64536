"""The native host calls and the Python path behind them: the same bits for the
calls both take, the Python path's errors and results for all others."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture
def both(monkeypatch):
    """f(call): the call's result with the native calls, checked against the one without them."""
    from ltx_amd import _lib

    _lib.lib()
    assert _lib.CALLS is not None, "ltx_amd/_calls.so is not built"
    native = _lib.CALLS

    def run(call):
        got = call()
        monkeypatch.setattr(_lib, "CALLS", None)
        want = call()
        monkeypatch.setattr(_lib, "CALLS", native)
        for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
            if b is None:
                assert a is None
                continue
            assert a.shape == b.shape and a.dtype == b.dtype and a.stride() == b.stride() and torch.equal(a, b)
        return got

    return run


def test_products(both):
    from ltx_amd.kernels import gemm

    g = torch.Generator(device=DEV).manual_seed(0)
    for m, k, n in ((1, 128, 8), (3, 1024, 72), (68, 2048, 264), (300, 512, 1032), (2300, 256, 4104)):
        w = gemm.make_weight(torch.randn(n, k, generator=g, device=DEV).bfloat16(),
                             torch.randn(n, generator=g, device=DEV), kind="mxfp4")
        x = torch.randn(m, k + 8, generator=g, device=DEV).bfloat16()[:, :k]
        res = torch.randn(m, n, generator=g, device=DEV).bfloat16()
        gate = torch.randn(n, generator=g, device=DEV)
        for rows in (x, gemm.quantize_rows_mxfp4(x)):
            for qlinear in (False, True):
                wt = gemm.LinearWeight("mxfp4", w.w, w.scale, w.bias, qlinear=qlinear)
                both(lambda: gemm.linear(rows, wt))
                both(lambda: gemm.linear(rows, wt, sigmoid_from=n - 5))
                both(lambda: gemm.linear(rows, wt, sigmoid_from=-3))
                both(lambda: gemm.linear(rows, wt, epilogue=gemm.EPI_GELU))
                for epi in (gemm.EPI_RESIDUAL, gemm.EPI_RESIDUAL_ROUND):
                    both(lambda: gemm.linear(rows, wt, epilogue=epi, residual=res, gate=gate))
            both(lambda: gemm.linear(rows, gemm.LinearWeight("mxfp4", w.w, w.scale)))
        both(lambda: gemm.linear(x[None], w))
        both(lambda: gemm.linear(x[0], w))
        both(lambda: gemm.linear(x[:1].expand(4, k), w))


def test_rows(both):
    from ltx_amd.kernels import gemm

    def pair(r):
        return r.codes, r.scales[:, :r.shape[0]].contiguous()

    for rows, k in ((1, 32), (5, 160), (130, 1024)):
        for dtype in (torch.bfloat16, torch.float16, torch.float32):
            x = torch.randn(rows, k + 16, device=DEV).to(dtype)[:, :k]
            both(lambda: pair(gemm.quantize_rows_mxfp4(x)))
            q = gemm.quantize_rows_mxfp4(x)
            both(lambda: gemm.dequantize_rows_mxfp4(q))
            both(lambda: pair(gemm.quantize_rows_mxfp4(x.view(1, *x.shape))))


def test_rotary(both):
    from ltx_amd.kernels import rope_ops

    inv, f = rope_ops.rotary_frequencies(32, scaling="yarn", stretch=4)
    for shape, kv in (((7, 4, 64), 2), ((2, 5, 3, 40), 3), ((1, 1, 32), 1)):
        q = torch.randn(shape, device=DEV).bfloat16()
        k = torch.randn(*shape[:-2], kv, shape[-1], device=DEV).bfloat16()
        lead = shape[:-2]
        for pos in (torch.arange(lead[-1], device=DEV), torch.rand(lead, device=DEV) * 9):
            for layout in rope_ops.ROTARY_LAYOUTS:
                kw = dict(layout=layout, factor=f)
                both(lambda: rope_ops.rotary(q, k, pos, inv, **kw))
                both(lambda: rope_ops.rotary(q, None, pos, inv, transpose=True, **kw))
                both(lambda: rope_ops.rotary(q.float(), k.float(), pos, inv, **kw))
                both(lambda: rope_ops.rotary(q[..., :1, :].expand(shape), k, pos, inv, **kw))


def test_what_the_native_calls_refuse_raises():
    from ltx_amd import _lib
    from ltx_amd.kernels import gemm, rope_ops

    w = gemm.make_weight(torch.randn(64, 128, device=DEV).bfloat16(), torch.zeros(64, device=DEV), kind="mxfp4")
    x = torch.randn(4, 128, device=DEV).bfloat16()
    for bad in (x[:, :64], x.cpu(), x.t()):
        with pytest.raises(ValueError):
            gemm.linear(bad, w)
    with pytest.raises(TypeError):
        gemm.linear(x.half(), w)
    with pytest.raises(ValueError):
        gemm.linear(x, gemm.LinearWeight("mxfp4", w.w, w.scale, w.bias.double()))
    with pytest.raises(ValueError):
        gemm.linear(x, gemm.LinearWeight("mxfp4", w.w, w.scale, w.bias[:32]))
    with pytest.raises(ValueError):
        gemm.linear(x, gemm.LinearWeight("mxfp4", w.w, w.scale[:, :60], w.bias))
    with pytest.raises(ValueError):
        gemm.linear(x, gemm.LinearWeight("mxfp4", w.w.cpu(), w.scale, w.bias))
    for kw in (dict(), dict(residual=x), dict(residual=x[:, :64], gate=torch.zeros(32, device=DEV))):
        with pytest.raises(ValueError):
            gemm.linear(x, w, epilogue=gemm.EPI_RESIDUAL, **kw)
    with pytest.raises(_lib.LtxKernelError):
        gemm.linear(x, w, epilogue=9)
    with pytest.raises(ValueError):
        gemm.dequantize_rows_mxfp4(gemm.Mx4Rows(w.w, w.scale[:, :60]))
    q, pos = torch.randn(4, 2, 64, device=DEV), torch.arange(4, device=DEV)
    inv, _ = rope_ops.rotary_frequencies(64)
    for a in ((q, None, pos[:3], inv), (q, q[:3], pos, inv), (q, None, pos.cpu(), inv), (q[..., ::2], None, pos, inv[:8]),
              (q, q.half(), pos, inv), (q[..., :32], None, pos, inv), (q.double(), None, pos, inv)):
        with pytest.raises(ValueError):
            rope_ops.rotary(*a)


def test_given_outputs(both):
    from ltx_amd.kernels import gemm, rope_ops

    g = torch.Generator(device=DEV).manual_seed(1)
    w = gemm.make_weight(torch.randn(72, 256, generator=g, device=DEV).bfloat16(), torch.zeros(72, device=DEV), kind="mxfp4")
    gate = torch.randn(72, generator=g, device=DEV)
    for m in (1, 5, 40):
        rows = torch.randn(m, 512, generator=g, device=DEV).bfloat16()
        x, out, res = rows[:, :256], rows[:, 256:328], rows[:, 336:408]
        want = gemm.linear(x, w, epilogue=gemm.EPI_RESIDUAL, residual=res, gate=gate)
        got = both(lambda: gemm.linear(x, w, epilogue=gemm.EPI_RESIDUAL, residual=res, gate=gate, out=out))
        assert got is out and torch.equal(out, want)
        keep = rows.clone()
        assert gemm.linear(x, w, epilogue=gemm.EPI_RESIDUAL, residual=res, gate=gate, out=res) is res  # in place
        assert torch.equal(res, want)
        keep[:, 336:408] = want
        assert torch.equal(rows, keep)  # and nothing beside it
        for bad in (rows[:, 192:264], rows[:, 328:400], out.float(), out[:, :64]):
            with pytest.raises(ValueError):
                gemm.linear(x, w, epilogue=gemm.EPI_RESIDUAL, residual=res, gate=gate, out=bad)

    inv, f = rope_ops.rotary_frequencies(64)
    for lead in ((1,), (9,), (2, 5)):
        buf = torch.randn(*lead, 10, 64, generator=g, device=DEV).bfloat16()
        q, k, rest = buf[..., :4, :], buf[..., 4:6, :], buf[..., 6:, :]
        pos = torch.arange(lead[-1], device=DEV)
        want = rope_ops.rotary(q, k, pos, inv)
        keep = buf.clone()
        got = both(lambda: rope_ops.rotary(q, k, pos, inv, out=(rest, None)))
        assert got[0] is rest and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        keep[..., 6:, :] = want[0]
        got = rope_ops.rotary(q, k, pos, inv, out=(q, k))
        keep[..., :4, :], keep[..., 4:6, :] = want
        assert got[0] is q and got[1] is k and torch.equal(buf, keep)
        for bad in ((buf[..., 1:5, :], k), (k, q), (q, buf[..., 3:5, :]), (q[..., :1, :].expand(q.shape), k)):
            with pytest.raises(ValueError):
                rope_ops.rotary(q, k, pos, inv, out=bad)
