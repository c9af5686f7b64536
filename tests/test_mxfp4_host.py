"""MXFP4 and rotary entry points on the host: refusals before any launch, the
scale-word helpers, the frequency stretches."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import quant as oq


@pytest.fixture(scope="module")
def lib():
    from ltx_amd import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("libltx_hip.so not built")
    return _lib.lib()


INVALID, UNSUPPORTED, ALIGN = -1, -2, -4


def test_quantiser_refusals(lib):
    def q(x=16, dtype=0, ldx=64, rows=4, k=64, codes=16, ldq=32, sc=16, lds=4):
        return lib.ltx_quantize_mxfp4(x, dtype, ldx, rows, k, codes, ldq, sc, lds, None)

    def d(codes=16, ldq=32, sc=16, lds=4, rows=4, k=64, out=16, ldo=64):
        return lib.ltx_dequantize_mxfp4_bf16(codes, ldq, sc, lds, rows, k, out, ldo, None)

    assert q(rows=0) == 0 and d(rows=0) == 0
    for f in (q, d):
        assert f(codes=None) == INVALID and f(sc=None) == INVALID and f(rows=-1) == INVALID
        assert f(k=48, ldq=32) == UNSUPPORTED  # not whole blocks
        assert f(ldq=16) == INVALID and f(lds=3) == INVALID
        assert f(codes=24) == ALIGN and f(sc=20) == ALIGN and f(ldq=40) == ALIGN and f(lds=6) == ALIGN
    assert q(x=None) == INVALID and q(dtype=3) == UNSUPPORTED and q(ldx=32) == INVALID
    assert q(x=24) == ALIGN and q(ldx=68) == ALIGN and q(ldx=66, dtype=2) == ALIGN
    assert d(out=None) == INVALID and d(ldo=32) == INVALID and d(ldo=66) == ALIGN and d(out=18) == ALIGN


def _gemm(lib, name, **over):
    a = dict(A=16, lda=256, As=16, ldas=8, W=16, ldw=128, Ws=16, ldws=64, bias=None, C=16, ldc=64, M=4, N=64, K=256,
             epi=0, R=None, ldr=0, gate=None, sig=64, ws=None, ws_bytes=0)
    a.update(over)
    head = (a["A"], a["lda"]) + ((a["As"], a["ldas"]) if "mx4" in name else ())
    return getattr(lib, name)(*head, a["W"], a["ldw"], a["Ws"], a["ldws"], a["bias"], a["C"], a["ldc"], a["M"],
                              a["N"], a["K"], a["epi"], a["R"], a["ldr"], a["gate"], a["sig"], a["ws"],
                              a["ws_bytes"], None)


@pytest.mark.parametrize("name", ["ltx_gemm_mxfp4_bf16", "ltx_gemm_mx4_bf16"])
def test_product_refusals(lib, name):
    def g(**over):
        return _gemm(lib, name, **over)

    assert g(M=0) == 0 and g(N=0) == 0
    for ptr in ("A", "W", "Ws", "C"):
        assert g(**{ptr: None}) == INVALID
        assert g(**{ptr: 24}) == ALIGN
    assert g(M=-1) == INVALID and g(N=-8) == INVALID and g(M=1 << 31) == UNSUPPORTED
    assert g(N=60) == UNSUPPORTED and g(K=224) == UNSUPPORTED and g(K=0) == UNSUPPORTED
    assert g(lda=64) == INVALID and g(ldw=112) == INVALID and g(ldc=56) == INVALID and g(ldws=60) == INVALID
    assert g(ldw=136) == ALIGN and g(ldc=68) == ALIGN and g(ldws=66) == ALIGN
    assert g(epi=5) == INVALID and g(epi=1 << 8) == INVALID and g(epi=1 << 13) == INVALID
    assert g(epi=2) == INVALID and g(epi=2, R=16, gate=16, ldr=56) == INVALID
    assert g(epi=2, R=16, gate=16, ldr=68) == ALIGN and g(epi=3, R=24, gate=16, ldr=64) == ALIGN
    assert g(bias=18) == ALIGN
    if "mx4" in name:
        assert g(As=None) == INVALID and g(As=24) == ALIGN and g(ldas=3) == INVALID and g(ldas=6) == ALIGN
        assert g(K=192, lda=96, ldw=96) == UNSUPPORTED
        assert g(M=1 << 26, ldas=1 << 26) == UNSUPPORTED  # 2^33 code bytes
    else:
        assert g(lda=260) == ALIGN


@pytest.mark.parametrize("name", ["ltx_gemm_mxfp4", "ltx_gemm_mx4"])
def test_workspace_sizes_and_refusals(lib, name):
    size = getattr(lib, name + "_workspace_bytes")
    assert size(-1, 8, 64) == -1 and size(0, 8, 64) == 0 and size(5, 0, 128) == 0
    seen = 0
    for m, n, k in ((1, 8, 16384), (68, 2048, 8192), (1, 4096, 4096), (33, 264, 4096), (6144, 16384, 4096)):
        need = size(m, n, k)
        assert need % (m * n * 4) == 0 and need // (m * n * 4) != 1
        if need:
            seen += 1
            kw = dict(M=m, N=n, K=k, lda=k, ldw=k // 2, ldws=-(-n // 4) * 4, ldas=-(-m // 4) * 4, ldc=n, sig=n)
            assert _gemm(lib, name + "_bf16", **kw) == INVALID
            assert _gemm(lib, name + "_bf16", ws=16, ws_bytes=need - 1, **kw) == INVALID
            assert _gemm(lib, name + "_bf16", ws=24, ws_bytes=need, **kw) == ALIGN
    assert seen


def test_rotary_refusals(lib):
    from ltx_amd import _lib

    def rows(x=16, out=16, heads=2, xt=128, ot=128):
        return _lib.RotaryRows(x, 0, xt, 64, out, 0, ot, 64, heads)

    def r(q=None, k=None, dtype=0, batch=1, tokens=3, dh=64, rot=64, pos=16, pt=0, pb=0, inv=16, flags=0, q_null=False):
        q = rows() if q is None else q
        return lib.ltx_rotary(None if q_null else ctypes.addressof(q), None if k is None else ctypes.addressof(k),
                              dtype, batch, tokens, dh, rot, pos, pt, pb, inv, 1.0, flags, None)

    assert r(tokens=0) == 0 and r(batch=0) == 0 and r(q=rows(heads=0)) == 0
    assert r(q_null=True) == INVALID and r(q=rows(x=None)) == INVALID and r(k=rows(out=None)) == INVALID
    assert r(rot=0) == INVALID and r(rot=7) == INVALID and r(rot=66) == INVALID and r(tokens=-1) == INVALID
    assert r(dtype=3) == UNSUPPORTED and r(pt=4) == UNSUPPORTED and r(dh=514, rot=64) == UNSUPPORTED
    assert r(flags=4) == INVALID and r(pos=None) == INVALID and r(inv=None) == INVALID and r(pb=-1) == INVALID
    assert r(pos=18) == ALIGN and r(pos=20, pt=1) == ALIGN and r(inv=20) == ALIGN and r(q=rows(x=17)) == ALIGN
    assert r(q=rows(heads=-1)) == INVALID


@pytest.mark.parametrize("rows,k", [(1, 32), (3, 160), (8, 256), (13, 512)])
def test_scale_word_helpers(rows, k):
    from ltx_amd.kernels import gemm

    rng = np.random.default_rng(rows)
    scales = rng.integers(0, 256, (rows, k // 32)).astype(np.uint8)
    _, want = oq.mxfp4_pack(np.zeros((rows, k), np.uint8), scales)
    words = gemm.mxfp4_scale_words(torch.from_numpy(scales))
    np.testing.assert_array_equal(words.numpy(), want)
    np.testing.assert_array_equal(gemm.mxfp4_block_scales(words, rows, k).numpy(), scales)


def test_python_refusals_without_a_gpu():
    from ltx_amd.kernels import gemm, rope_ops

    codes, words = torch.zeros(8, 64, dtype=torch.uint8), torch.zeros(1, 8, dtype=torch.int32)
    w = gemm.LinearWeight("mxfp4", codes, words)
    assert w.in_features == 128 and w.out_features == 8
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError):  # host tensors
        gemm.linear(x, w)
    with pytest.raises(TypeError):
        gemm.linear(x.float(), w)
    with pytest.raises(ValueError):
        gemm.linear(x[:, :64], w)
    with pytest.raises(ValueError):
        gemm.linear(x, w, tile=gemm.TILE_128)
    with pytest.raises(ValueError):
        gemm.linear(x, w, splits=2)
    with pytest.raises(ValueError):
        gemm.linear(gemm.MxRows(codes, words), w)
    with pytest.raises(ValueError):
        gemm.linear(gemm.Mx4Rows(codes, words), gemm.LinearWeight("mxfp8", codes, words))
    with pytest.raises(ValueError):  # too few scale words
        gemm.linear(x, gemm.LinearWeight("mxfp4", codes, words[:, :4]))
    with pytest.raises(ValueError):
        gemm.linear(x, w, out=torch.zeros(2, 16, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        gemm.quantize_rows_mxfp4(torch.zeros(2, 48))
    with pytest.raises(TypeError):
        gemm.quantize_rows_mxfp4(torch.zeros(2, 64, dtype=torch.float64))

    q, pos = torch.zeros(5, 4, 64, dtype=torch.bfloat16), torch.arange(5)
    inv, _ = rope_ops.rotary_frequencies(64, device="cpu")
    for kw in (dict(layout="quarter"), dict(out=(q.float(), None)), dict(out=(q, q)),
               dict(out=(q[:, :1].expand(5, 4, 64), None))):
        with pytest.raises(ValueError):
            rope_ops.rotary(q, None, pos, inv, **kw)
    for a in ((q[0], None, pos, inv), (q, q[:4], pos, inv), (q, q[..., :32], pos, inv), (q, None, pos[:4], inv),
              (q, None, pos.half(), inv), (q, None, pos, inv.float()), (q[..., :32], None, pos, inv),
              (q, None, pos, inv)):
        with pytest.raises(ValueError):
            rope_ops.rotary(*a)


def test_frequency_stretches():
    from ltx_amd.kernels.rope_ops import rotary_frequencies

    d, theta = 64, 10000.0
    base, f = rotary_frequencies(d, theta, device="cpu")
    np.testing.assert_allclose(base.numpy(), theta ** (-np.arange(0, d, 2) / d), rtol=1e-14)
    assert f == 1.0
    lin, f = rotary_frequencies(d, theta, scaling="linear", stretch=8, device="cpu")
    np.testing.assert_allclose(lin.numpy(), base.numpy() / 8, rtol=1e-14)
    ntk, f = rotary_frequencies(d, theta, scaling="ntk", stretch=8, device="cpu")
    assert abs(ntk[0].item() - 1) < 1e-12 and abs(ntk[-1].item() * 8 / base[-1].item() - 1) < 1e-9 and f == 1.0
    yarn, f = rotary_frequencies(d, theta, scaling="yarn", stretch=16, original_length=4096, device="cpu")
    assert f == pytest.approx(0.1 * math.log(16) + 1)
    turns = 4096 * base.numpy() / (2 * math.pi)
    r = yarn.numpy() / base.numpy()
    np.testing.assert_allclose(r[turns > 45], 1.0, rtol=1e-12)  # one pair beyond the borders' rounding outwards
    np.testing.assert_allclose(r[turns < 0.7], 1 / 16, rtol=1e-12)
    assert ((r >= 1 / 16 - 1e-12) & (r <= 1 + 1e-12)).all() and (np.diff(r) <= 1e-12).all()
    same, f = rotary_frequencies(d, theta, scaling="yarn", stretch=1, device="cpu")
    assert torch.equal(same, base) and f == 1.0
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling="x"),
                dict(rotary_dim=8, theta=1.0), dict(rotary_dim=8, stretch=0.5)):
        with pytest.raises(ValueError):
            rotary_frequencies(device="cpu", **bad)


def test_overlapping_outputs_are_refused():
    from ltx_amd import _lib
    from ltx_amd.kernels import gemm, rope_ops

    rng = np.random.default_rng(3)
    for _ in range(300):  # the rule against the sets of addresses
        base = torch.zeros(400, dtype=torch.bfloat16)
        views = []
        for _ in range(2):
            sizes = [int(v) for v in rng.integers(1, 5, 3)]
            strides = [int(v) for v in rng.choice([0, 1, 2, 3, 8, 16, 32, 33], 3)]
            views.append(base.as_strided(sizes, strides, int(rng.integers(0, 60))))
        a, b = views
        at = [torch.arange(400).as_strided(v.shape, v.stride(), v.storage_offset()).flatten().tolist() for v in views]
        if set(at[0]) & set(at[1]):
            assert _lib.overlaps(a, b) and _lib.overlaps(b, a)
        if len(set(at[0])) < len(at[0]):
            assert _lib.self_overlaps(a)
    buf = torch.zeros(2, 5, 12, 64, dtype=torch.bfloat16)
    q, k, rest = buf[:, :, :4], buf[:, :, 4:6], buf[:, :, 6:]
    assert not _lib.overlaps(q, k) and not _lib.overlaps(rest, q) and not _lib.overlaps(buf[0], buf[1])
    assert not _lib.overlaps(buf[..., :32], buf[..., 32:]) and _lib.overlaps(buf[..., :33], buf[..., 32:])
    assert not _lib.self_overlaps(q) and not _lib.self_overlaps(buf.transpose(1, 2)) and _lib.self_overlaps(q[:, :1].expand_as(q))

    pos = torch.arange(5)
    inv, _ = rope_ops.rotary_frequencies(64, device="cpu")
    for out in ((k.clone(), q.clone()), (buf[:, :, 1:5], k), (q, buf[:, :, 3:5]), (buf[:, :, 6:10], buf[:, :, 9:11]),
                (q.transpose(1, 2).reshape(-1).as_strided(q.shape, (0, 256, 64, 1)), None)):
        with pytest.raises(ValueError):
            rope_ops.rotary(q, k, pos, inv, out=out)
    for out in ((q, k), (rest[:, :, :4], rest[:, :, 4:]), (torch.empty_like(q), None)):
        with pytest.raises(ValueError, match="on one GPU"):  # nothing to object to but the host's memory
            rope_ops.rotary(q, k, pos, inv, out=out)

    w = gemm.LinearWeight("mxfp4", torch.zeros(128, 64, dtype=torch.uint8), torch.zeros(1, 128, dtype=torch.int32))
    rows = torch.zeros(6, 256, dtype=torch.bfloat16)
    gate = torch.zeros(128)
    x = rows[:4, :128]
    res = dict(epilogue=gemm.EPI_RESIDUAL, gate=gate)
    for kw in (dict(out=x), dict(out=rows[1:5, :128]), dict(out=rows[:4, 64:192]),
               dict(out=rows[:4, 128:], residual=rows[1:5, 128:], **res)):
        with pytest.raises(ValueError, match="overlaps"):
            gemm.linear(x, w, **kw)
    for kw in (dict(out=rows[:4, 128:]), dict(out=rows[:4, 128:], residual=rows[:4, 128:], **res)):
        with pytest.raises(ValueError, match="on one GPU"):
            gemm.linear(x, w, **kw)


def test_rows_of_no_elements_are_refused():
    from ltx_amd.kernels import gemm

    codes, words = torch.zeros(8, 0, dtype=torch.uint8), torch.zeros(0, 8, dtype=torch.int32)
    with pytest.raises(ValueError):
        gemm.quantize_rows_mxfp4(torch.zeros(5, 0))
    with pytest.raises(ValueError):
        gemm.dequantize_rows_mxfp4(gemm.Mx4Rows(codes, words))
    for x in (torch.zeros(2, 5, 0, dtype=torch.bfloat16), gemm.Mx4Rows(codes, words)):
        with pytest.raises(ValueError):
            gemm.linear(x, gemm.LinearWeight("mxfp4", codes, words))


@pytest.mark.parametrize("name", ["ltx_gemm_mxfp4_bf16", "ltx_gemm_mx4_bf16"])
def test_products_past_one_launch_are_refused(lib, name):
    """More threads than one launch has, or strides that overflow a byte offset."""
    m, n = 1 << 28, 1 << 28
    assert _gemm(lib, name, M=m, ldas=m) == UNSUPPORTED
    assert _gemm(lib, name, N=n, ldc=n, ldws=n, sig=n) == UNSUPPORTED
    m, n = 1 << 18, 1 << 17
    assert _gemm(lib, name, M=m, ldas=m, N=n, ldc=n, ldws=n, sig=n) == UNSUPPORTED
    for stride in ("lda", "ldw", "ldc", "ldws"):
        assert _gemm(lib, name, M=1, **{stride: 1 << 62}) == UNSUPPORTED


def test_rows_past_one_launch_are_refused(lib):
    from ltx_amd import _lib

    k, rows = 512, 1 << 28
    assert lib.ltx_quantize_mxfp4(16, 0, k, rows, k, 16, k // 2, 16, rows, None) == UNSUPPORTED
    assert lib.ltx_dequantize_mxfp4_bf16(16, k // 2, 16, rows, rows, k, 16, k, None) == UNSUPPORTED
    q = _lib.RotaryRows(16, 0, 64, 64, 16, 0, 64, 64, 1)
    assert lib.ltx_rotary(ctypes.addressof(q), None, 0, 1, 1 << 27, 64, 64, 16, 0, 0, 16, 1.0, 0, None) == UNSUPPORTED
