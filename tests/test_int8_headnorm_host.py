"""int8 products and the per-head norm on the host: refusals before any launch."""

from __future__ import annotations

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from ltx_amd import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("libltx_hip.so not built")
    return _lib.lib()


INVALID, UNSUPPORTED, ALIGN = -1, -2, -4


def test_row_quantiser_refusals(lib):
    def q(x=16, dtype=0, ldx=64, rows=4, k=64, codes=16, ldq=64, sc=4):
        return lib.ltx_quantize_int8(x, dtype, ldx, rows, k, codes, ldq, sc, None)

    assert q(rows=0) == 0
    assert q(x=None) == INVALID and q(codes=None) == INVALID and q(sc=None) == INVALID and q(rows=-1) == INVALID
    assert q(ldx=48) == INVALID and q(ldq=48) == INVALID
    assert q(dtype=3) == UNSUPPORTED and q(k=56) == UNSUPPORTED and q(rows=1 << 24) == UNSUPPORTED
    assert q(x=24) == ALIGN and q(codes=24) == ALIGN and q(sc=6) == ALIGN and q(ldx=68) == ALIGN and q(ldq=72) == ALIGN
    assert q(dtype=2, ldx=66) == ALIGN
    assert lib.ltx_dequantize_w8_bf16(16, 512, 16, 1 << 28, 512, 16, 512, None) == UNSUPPORTED


def _gemm(lib, **over):
    a = dict(A=16, lda=256, sa=4, W=16, ldw=256, sw=4, bias=None, C=16, ldc=64, M=4, N=64, K=256, epi=0, R=None, ldr=0,
             gate=None, sig=64, ws=None, ws_bytes=0)
    a.update(over)
    return lib.ltx_gemm_i8_bf16(a["A"], a["lda"], a["sa"], a["W"], a["ldw"], a["sw"], a["bias"], a["C"], a["ldc"], a["M"],
                                a["N"], a["K"], a["epi"], a["R"], a["ldr"], a["gate"], a["sig"], a["ws"], a["ws_bytes"],
                                None)


def test_product_refusals(lib):
    def g(**over):
        return _gemm(lib, **over)

    assert g(M=0) == 0 and g(N=0) == 0
    for ptr in ("A", "W", "C", "sa", "sw"):
        assert g(**{ptr: None}) == INVALID
    for ptr in ("A", "W", "C"):
        assert g(**{ptr: 24}) == ALIGN
    for ptr in ("sa", "sw", "bias"):
        assert g(**{ptr: 18}) == ALIGN
    assert g(M=-1) == INVALID and g(N=-8) == INVALID and g(K=-64) == INVALID
    assert g(N=60) == UNSUPPORTED and g(K=224) == UNSUPPORTED and g(K=0) == UNSUPPORTED
    assert g(K=1 << 17, lda=1 << 17, ldw=1 << 17) == UNSUPPORTED  # sums past 31 bits
    assert g(lda=240) == INVALID and g(ldw=240) == INVALID and g(ldc=56) == INVALID
    assert g(lda=264) == ALIGN and g(ldw=264) == ALIGN and g(ldc=68) == ALIGN
    assert g(epi=5) == INVALID and g(epi=1 << 8) == INVALID and g(epi=1 << 13) == INVALID
    assert g(epi=2) == INVALID and g(epi=2, R=16, gate=16, ldr=56) == INVALID
    assert g(epi=2, R=16, gate=16, ldr=68) == ALIGN and g(epi=3, R=24, gate=16, ldr=64) == ALIGN
    for stride in ("lda", "ldw", "ldc"):
        assert g(M=1, **{stride: 1 << 62}) == UNSUPPORTED
    big = 1 << 28
    assert g(M=big) == UNSUPPORTED and g(N=big, ldc=big, sig=big) == UNSUPPORTED
    assert g(M=1 << 18, N=1 << 17, ldc=1 << 17, sig=1 << 17) == UNSUPPORTED


def test_workspace_sizes_and_refusals(lib):
    size = lib.ltx_gemm_i8_workspace_bytes
    assert size(-1, 8, 64) == -1 and size(0, 8, 64) == 0 and size(5, 0, 64) == 0 and size(5, 8, 0) == 0
    for m, n, k in ((1, 8, 16384), (68, 2048, 8192), (130, 512, 16384), (1, 4096, 4096), (33, 264, 4096),
                    (200, 256, 65536), (6144, 16384, 4096)):
        need = size(m, n, k)
        assert need >= 0 and need % (m * n * 4) == 0 and need // (m * n * 4) != 1
        if need:
            kw = dict(M=m, N=n, K=k, lda=k, ldw=k, ldc=n, sig=n)
            assert _gemm(lib, **kw) == INVALID
            assert _gemm(lib, ws=16, ws_bytes=need - 1, **kw) == INVALID
            assert _gemm(lib, ws=24, ws_bytes=need, **kw) == ALIGN


def test_headnorm_refusals(lib):
    from ltx_amd import _lib

    def rows(x=16, out=16, g=16, w=16, dw=None, heads=2):
        return _lib.HeadnormRows(x, 0, 128, 64, out, 0, 128, 64, g, 0, 128, 64, w, dw, heads)

    def both(**kw):
        return f(**kw), b(**kw)

    def f(q=None, k=None, dtype=0, batch=1, tokens=3, dh=64, rot=64, pos=16, pt=0, pb=0, inv=16, eps=0.0, flags=0,
          q_null=False, **_):
        q = rows() if q is None else q
        return lib.ltx_headnorm_rotary(None if q_null else ctypes.addressof(q), None if k is None else ctypes.addressof(k),
                                       dtype, batch, tokens, dh, rot, pos, pt, pb, inv, 1.0, eps, 0.0, flags, None)

    def b(q=None, k=None, dtype=0, batch=1, tokens=3, dh=64, rot=64, pos=16, pt=0, pb=0, inv=16, eps=0.0, flags=0,
          q_null=False, ws=None, ws_bytes=0):
        q = rows() if q is None else q
        return lib.ltx_headnorm_rotary_grad(None if q_null else ctypes.addressof(q),
                                            None if k is None else ctypes.addressof(k), dtype, batch, tokens, dh, rot, pos,
                                            pt, pb, inv, 1.0, eps, 0.0, flags, ws, ws_bytes, None)

    for kw, want in ((dict(tokens=0), 0), (dict(batch=0), 0), (dict(q=rows(heads=0)), 0), (dict(q_null=True), INVALID),
                     (dict(q=rows(x=None)), INVALID), (dict(k=rows(out=None)), INVALID), (dict(rot=-2), INVALID),
                     (dict(rot=7), INVALID), (dict(rot=66), INVALID), (dict(tokens=-1), INVALID), (dict(dtype=3), UNSUPPORTED),
                     (dict(pt=4), UNSUPPORTED), (dict(dh=514), UNSUPPORTED), (dict(dh=0, rot=0), INVALID),
                     (dict(flags=2), INVALID), (dict(pos=None), INVALID), (dict(inv=None), INVALID), (dict(pb=-1), INVALID),
                     (dict(pos=18), ALIGN), (dict(pos=20, pt=1), ALIGN), (dict(inv=20), ALIGN), (dict(q=rows(x=17)), ALIGN),
                     (dict(q=rows(w=18)), ALIGN), (dict(q=rows(heads=-1)), INVALID), (dict(eps=-1.0), INVALID),
                     (dict(eps=float("nan")), INVALID), (dict(q=rows(heads=(1 << 30) + 1)), UNSUPPORTED),
                     (dict(tokens=1 << 27), UNSUPPORTED)):
        assert both(**kw) == (want, want), kw
    assert b(q=rows(g=None)) == INVALID and b(q=rows(g=17)) == ALIGN
    assert b(q=rows(w=None, dw=16)) == INVALID and b(q=rows(dw=18)) == ALIGN
    need = lib.ltx_headnorm_rotary_grad_workspace_bytes(64)
    assert need > 0 and lib.ltx_headnorm_rotary_grad_workspace_bytes(-1) == -1
    assert b(q=rows(dw=16)) == INVALID and b(q=rows(dw=16), ws=16, ws_bytes=need - 1) == INVALID
    assert b(q=rows(dw=16), ws=18, ws_bytes=need) == ALIGN


def test_python_refusals_without_a_gpu():
    from ltx_amd.kernels import gemm

    codes, scales = torch.zeros(8, 128, dtype=torch.int8), torch.zeros(8)
    w = gemm.LinearWeight("int8", codes, scales)
    rows = gemm.Int8Rows(torch.zeros(2, 128, dtype=torch.int8), torch.zeros(2))
    assert rows.shape == (2, 128)
    with pytest.raises(ValueError, match="on one GPU"):
        gemm.linear(rows, w)
    with pytest.raises(ValueError, match="on one GPU"):
        gemm.dequantize_rows_int8(rows)
    with pytest.raises(ValueError, match="on one GPU"):
        gemm.quantize_rows_int8(torch.zeros(2, 64))
    for kind in ("bf16", "mxfp8", "mxfp4"):
        with pytest.raises(ValueError, match="do not go with"):
            gemm.linear(rows, gemm.LinearWeight(kind, codes, scales))
    for kw in (dict(tile=gemm.TILE_128), dict(splits=2), dict(out=torch.zeros(2, 16, dtype=torch.bfloat16)),
               dict(out=torch.zeros(2, 8)), dict(epilogue=gemm.EPI_RESIDUAL),
               dict(epilogue=gemm.EPI_RESIDUAL, residual=torch.zeros(2, 8, dtype=torch.bfloat16), gate=torch.zeros(7)),
               dict(epilogue=gemm.EPI_RESIDUAL, residual=torch.zeros(2, 8), gate=torch.zeros(8))):
        with pytest.raises(ValueError):
            gemm.linear(rows, w, **kw)
    for bad in (gemm.Int8Rows(rows.codes, torch.zeros(3)), gemm.Int8Rows(rows.codes, torch.zeros(2, 1)),
                gemm.Int8Rows(rows.codes.byte(), rows.scales), gemm.Int8Rows(rows.codes, rows.scales.double()),
                gemm.Int8Rows(rows.codes, torch.zeros(4)[::2]), gemm.Int8Rows(rows.codes[:, :64], rows.scales),
                gemm.Int8Rows(torch.zeros(128, 2, dtype=torch.int8).T, rows.scales),
                gemm.Int8Rows(rows.codes[:1].expand(2, 128), rows.scales), gemm.Int8Rows(rows.codes[:, :0], rows.scales)):
        with pytest.raises(ValueError):
            gemm.linear(bad, w)
    for x in (torch.zeros(2, 24), torch.zeros(5, 0)):
        with pytest.raises(ValueError):
            gemm.quantize_rows_int8(x)
    with pytest.raises(TypeError):
        gemm.quantize_rows_int8(torch.zeros(2, 64, dtype=torch.float64))
    # outputs over operands
    buf = torch.zeros(6, 512, dtype=torch.bfloat16)
    inside = buf.view(torch.int8)
    wide = gemm.LinearWeight("int8", torch.zeros(128, 128, dtype=torch.int8), torch.zeros(128))
    over = gemm.Int8Rows(inside[:4, :128], torch.zeros(4))
    res = dict(epilogue=gemm.EPI_RESIDUAL, gate=torch.zeros(128))
    for kw in (dict(out=buf[:4, :128]), dict(out=buf[:4, 128:256], residual=buf[1:5, 128:256], **res)):
        with pytest.raises(ValueError, match="overlaps"):
            gemm.linear(over, wide, **kw)
    for kw in (dict(out=buf[:4, 128:256]), dict(out=buf[:4, 128:256], residual=buf[:4, 128:256], **res)):
        with pytest.raises(ValueError, match="on one GPU"):
            gemm.linear(over, wide, **kw)


def test_headnorm_python_refusals_without_a_gpu():
    from ltx_amd.kernels import rope_ops

    buf = torch.zeros(2, 5, 12, 64, dtype=torch.bfloat16)
    q, k, rest = buf[:, :, :4], buf[:, :, 4:6], buf[:, :, 6:]
    pos, w = torch.arange(5), torch.zeros(64)
    inv, _ = rope_ops.rotary_frequencies(64, device="cpu")
    f, b = rope_ops.headnorm_rotary, rope_ops.headnorm_rotary_grad
    gq, gk = torch.zeros_like(q), torch.zeros_like(k)
    for a in ((q[0, 0], None, None, None, pos, inv), (q, k[..., :32], w, w, pos, inv), (q, k[:1], w, w, pos, inv),
              (q, k.float(), w, w, pos, inv), (q.double(), None, w, None, pos, inv), (q, None, w, w, pos, inv),
              (q, k, w[:32], w, pos, inv), (q, k, w.bfloat16(), w, pos, inv), (q, k, w, torch.zeros(128)[::2], pos, inv),
              (q, k, w, w, pos[:4], inv), (q, k, w, w, pos.half(), inv), (q, k, w, w, pos, inv.float()),
              (q, k, w, w, pos, None), (q, k, w, w, None, inv), (q[..., :32], None, w[:32], None, pos, inv),
              (torch.zeros(5, 64, 4).transpose(1, 2), None, None, None, pos, inv)):
        with pytest.raises(ValueError, match="(?!.*on one GPU)"):
            f(*a)
    for kw in (dict(layout="quarter"), dict(eps=-1.0), dict(out=(q.float(), None)), dict(out=(q, q)),
               dict(out=(k, q)), dict(out=(buf[:, :, 1:5], k)), dict(out=(q, buf[:, :, 3:5])),
               dict(out=(q[:, :1].expand(2, 5, 4, 64), None)), dict(out=(rest[:, :, :4], rest[:, :, 3:5]))):
        with pytest.raises(ValueError) as e:
            f(q, k, w, w, pos, inv, **kw)
        assert "on one GPU" not in str(e.value), kw
    with pytest.raises(ValueError, match="factor"):
        f(q, k, w, w, None, None, factor=2.0)
    with pytest.raises(ValueError, match="there is no k"):
        f(q, None, w, None, pos, inv, out=(q, k))
    for out in (None, (q, k), (rest[:, :, :4], rest[:, :, 4:]), (torch.empty_like(q), None)):
        with pytest.raises(ValueError, match="on one GPU"):  # nothing to object to but the host's memory
            f(q, k, w, w, pos, inv, out=out)
    for a in ((None, None, q, None), (gq[:1], gk, q, k), (gq, None, q, k), (gq.float(), gk, q, k), (gq, gk, q, None)):
        with pytest.raises(ValueError) as e:
            b(*a, w, w if a[3] is not None else None, pos, inv)
        assert "on one GPU" not in str(e.value), a
    for out in ((k, q), (gk, gq), (gq, gq[:, :, :2]), (rest[:, :, :4], q[:, :, :2])):
        with pytest.raises(ValueError) as e:
            b(gq, gk, q, k, w, w, pos, inv, out=out)
        assert "on one GPU" not in str(e.value), out
    for out in (None, (gq, gk), (q, k), (gq, k), (rest[:, :, :4], None)):
        with pytest.raises(ValueError, match="on one GPU"):
            b(gq, gk, q, k, w, w, pos, inv, out=out)
