"""MXFP4 quantisation and products against float64.

Quantisation is exact: codes and scales equal the oracle's, bit for bit.

Products: the decoded operands are exact in bf16, their products exact in
fp32, so what a result may differ by is the fp32 accumulation and the stated
roundings.  K additions, each off by at most one unit of 2^-23 of the running
sum (the matrix pipe may truncate), stay within K 2^-23 sum |a w| = A; a bf16
rounding is off by at most 2^-8 of the value.  GELU's slope is at most 1.13 and
the sigmoid's 1/4; their hardware exp and reciprocal are off by 2e-6 at most.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import quant as oq

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = 2.0 ** -8


def _codes_words(rows: int, k: int, seed: int, spread: int = 6):
    """Random stored MXFP4 rows and their float64 values (on the GPU)."""
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 16, (rows, k)).astype(np.uint8)
    scales = rng.integers(120 - spread, 121 + spread, (rows, k // 32)).astype(np.uint8)
    b, w = oq.mxfp4_pack(codes, scales)
    return (torch.from_numpy(b).to(DEV), torch.from_numpy(w).to(DEV),
            torch.from_numpy(oq.mxfp4_dequantize(codes, scales)).to(DEV))


def _reference(x, w, bias, epi, res, gate, sig, rtb):
    """float64 result and the largest error that the module text allows."""
    acc = x @ w.T
    a = w.shape[1] * 2.0 ** -23 * (x.abs() @ w.abs().T)
    y, e = acc, a
    if rtb:
        e = e + HALF * acc.abs()
    if bias is not None:
        y = y + bias.double()
        e = e + 2.0 ** -23 * y.abs()
    out, err = y, e
    if epi == "gelu":
        out = torch.nn.functional.gelu(y, approximate="tanh")
        err = 1.13 * e + 2e-6 * (1 + y.abs())
    elif epi == "sigmoid2":
        out, err = 2 * torch.sigmoid(y), e / 2 + 4e-6
    elif epi.startswith("residual"):
        eb = e + HALF * (y.abs() + e)  # the branch, rounded
        prod = gate.double() * y
        ep = gate.double().abs() * eb
        if epi == "residual_round":
            ep = ep + HALF * (prod.abs() + ep)
        out, err = res.double() + prod, ep + 2.0 ** -22 * (res.double().abs() + prod.abs())
    if sig is not None:
        out, err = out.clone(), err.clone()
        out[:, sig:], err[:, sig:] = 2 * torch.sigmoid(y[:, sig:]), e[:, sig:] / 2 + 4e-6
    return out, err + HALF * (out.abs() + err)


def _check(got, ref, err):
    torch.cuda.synchronize()
    over = (got.double() - ref).abs() - err
    assert torch.isfinite(got).all()
    assert over.max().item() <= 0, (over.max().item(), (got.double() - ref).abs().max().item())


EPI = {"bias": 0, "gelu": 1, "residual": 2, "residual_round": 3, "sigmoid2": 4}
# (M, K, N): one row to tiles of every height, ragged in each direction, depths of a half scale word, of one
# word, of no whole stage, long ones
SHAPES = [(1, 64, 8), (1, 4096, 4096), (2, 16384, 24), (5, 192, 40), (15, 448, 136), (16, 2048, 264),
          (17, 128, 8), (33, 320, 136), (64, 832, 72), (65, 1024, 2056), (68, 2048, 8192), (68, 8192, 2048),
          (121, 4096, 520), (129, 576, 1000), (256, 4096, 1024), (300, 1024, 712), (700, 2048, 520),
          (1296, 512, 2064), (1296, 704, 4096), (257, 16384, 264), (2049, 256, 4104), (3456, 640, 4096)]
MX_SHAPES = [s for s in SHAPES if s[1] % 128 == 0] + [(3, 256, 16), (31, 384, 128), (130, 1152, 264),
                                                    (5000, 384, 2056), (4097, 1280, 2568)]


def _epilogues(m, n):
    pick = (m + n) % 5
    return sorted({"bias", list(EPI)[pick]})


def _run(x, wt, epi, res, gate, sig):
    from ltx_amd.kernels import gemm

    return gemm.linear(x, wt, epilogue=EPI[epi], residual=res, gate=gate, sigmoid_from=sig)


@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("m,k,n", SHAPES + [s for s in MX_SHAPES if s not in SHAPES])
def test_products(m, k, n, quantised):
    from ltx_amd.kernels import gemm

    if quantised and (m, k, n) not in MX_SHAPES:
        pytest.skip("K is no multiple of 128")
    print(f"mxfp4 product M={m} K={k} N={n} quantised={quantised}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(m + 3 * k + 7 * n)
    wc, ws, w = _codes_words(n, k, seed=n + k)
    bias = torch.randn(n, generator=g, device=DEV)
    if quantised:
        xc, xs, xv = _codes_words(m, k, seed=m)
        x = gemm.Mx4Rows(xc, xs)
    else:
        x = torch.randn(m, k, generator=g, device=DEV).bfloat16()
        xv = x.double()
    for epi in _epilogues(m, n):
        res = gate = None
        if epi.startswith("residual"):
            res = torch.randn(m, n, generator=g, device=DEV).bfloat16()
            gate = torch.randn(n, generator=g, device=DEV)
        for qlinear in (False, True):
            wt = gemm.LinearWeight("mxfp4", wc, ws, bias, qlinear=qlinear)
            sig = None if epi != "bias" or not qlinear else max(n - 12, 4)
            print(f"  {epi} qlinear={qlinear} sig={sig}", flush=True)
            got = _run(x, wt, epi, res, gate, sig)
            _check(got, *_reference(xv, w, bias, epi, res, gate, sig, qlinear))


@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("m,k,n", [(3, 1152, 72), (200, 640, 392), (1800, 1024, 4096)])
def test_strided_operands_and_what_lies_beside_them(m, k, n, quantised):
    """Row-strided activations, codes, residual and output, wider scale words;
    nothing outside the output's rows and columns changes, and no bias."""
    from ltx_amd.kernels import gemm

    print(f"mxfp4 strided M={m} K={k} N={n} quantised={quantised}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(m)
    wc, ws, w = _codes_words(n, k, seed=5)
    wide = torch.full((n, k // 2 + 48), 255, dtype=torch.uint8, device=DEV)
    wide[:, 16:16 + k // 2] = wc
    words = torch.full((ws.shape[0] + 1, ws.shape[1] + 8), -1, dtype=torch.int32, device=DEV)
    words[:ws.shape[0], 4:4 + ws.shape[1]] = ws
    wt = gemm.LinearWeight("mxfp4", wide[:, 16:16 + k // 2], words[:ws.shape[0], 4:], None)
    if quantised:
        xc, xs, xv = _codes_words(m, k, seed=m)
        xw = torch.full((m, k // 2 + 16), 255, dtype=torch.uint8, device=DEV)
        xw[:, :k // 2] = xc
        x = gemm.Mx4Rows(xw[:, :k // 2], xs)
    else:
        buf = torch.full((m, k + 24), float("nan"), dtype=torch.bfloat16, device=DEV)
        buf[:, 8:8 + k] = torch.randn(m, k, generator=g, device=DEV).bfloat16()
        x = buf[:, 8:8 + k]
        xv = x.double()
    whole = torch.full((m + 2, n + 16), 7.0, dtype=torch.bfloat16, device=DEV)
    res = torch.randn(m, n + 8, generator=g, device=DEV).bfloat16()[:, :n]
    gate = torch.randn(n, generator=g, device=DEV)
    got = gemm.linear(x, wt, epilogue=gemm.EPI_RESIDUAL, residual=res, gate=gate, out=whole[1:m + 1, 8:8 + n])
    _check(got, *_reference(xv, w, None, "residual", res, gate, None, False))
    outside = whole.clone()
    outside[1:m + 1, 8:8 + n] = 7.0
    assert (outside == 7.0).all()
    # in place on the residual
    inplace = res.clone()
    gemm.linear(x, wt, epilogue=gemm.EPI_RESIDUAL, residual=inplace, gate=gate, out=inplace)
    assert torch.equal(inplace, got)


@pytest.mark.parametrize("rows,stride,k,n", [(2100, 1 << 19, 256, 264), (150, 1 << 23, 512, 136), (40, 1 << 25, 320, 72)])
def test_activations_past_two_gib(rows, stride, k, n):
    """Rows so far apart that byte offsets pass 31 and 32 bits: the product goes
    in pieces of rows, or to the kernel with 64-bit addresses."""
    from ltx_amd.kernels import gemm

    buf = torch.empty(rows, stride, dtype=torch.bfloat16, device=DEV)
    x = buf[:, :k]
    g = torch.Generator(device=DEV).manual_seed(8)
    x.copy_(torch.randn(rows, k, generator=g, device=DEV))
    wc, ws, w = _codes_words(n, k, seed=2)
    got = gemm.linear(x, gemm.LinearWeight("mxfp4", wc, ws))
    _check(got, *_reference(x.double(), w, None, "bias", None, None, None, False))


@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("m,n", [(1, 64), (90, 200), (2000, 4096)])
def test_non_finite_rows_and_columns_stay_theirs(m, n, quantised):
    """A NaN scale spoils its column (weights) or row (activations), an infinite
    activation its row; every other value is what it is without them."""
    from ltx_amd.kernels import gemm

    k = 768
    wc, ws, _ = _codes_words(n, k, seed=1)
    g = torch.Generator(device=DEV).manual_seed(2)
    if quantised:
        xc, xs, _ = _codes_words(m, k, seed=3)
        x = gemm.Mx4Rows(xc, xs)
    else:
        x = torch.randn(m, k, generator=g, device=DEV).bfloat16()
    clean = gemm.linear(x, gemm.LinearWeight("mxfp4", wc, ws))
    bad_w = ws.clone()
    bad_w[2, n // 2] |= 0xff00
    row = m // 2
    if quantised:
        bad_s = xs.clone()
        bad_s[1, row] |= 0xff
        bad = gemm.Mx4Rows(xc, bad_s)
    else:
        bad = x.clone()
        bad[row, 5] = float("inf")
    got = gemm.linear(bad, gemm.LinearWeight("mxfp4", wc, bad_w))
    torch.cuda.synchronize()
    assert not torch.isfinite(got[row]).any() or not quantised
    assert torch.isnan(got[:, n // 2]).all()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[row], keep[:, n // 2] = False, False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 160), (17, 512), (130, 672), (1000, 1024)])
def test_quantiser_equals_the_rule(rows, k, dtype):
    """Random bit patterns (every exponent, subnormals, NaN and infinities in
    some blocks) and ties: codes, scale bytes and decoded values."""
    from ltx_amd.kernels import gemm

    rng = np.random.default_rng(rows + k)
    if dtype == torch.float32:
        x = torch.from_numpy(rng.integers(0, 1 << 32, (rows, k), dtype=np.uint64).astype(np.uint32).view(np.float32))
    else:
        x = torch.from_numpy(rng.integers(0, 1 << 16, (rows, k)).astype(np.uint16).view(np.int16)).view(dtype)
    x = x.clone()
    blocks = x.view(rows, k // 32, 32)
    kind = torch.from_numpy(rng.integers(0, 8, (rows, k // 32)))
    # of eight blocks: one as it is, one of zeros, one of ties (quarter steps below 8, random power), the
    # others finite values of a few octaves
    mag = torch.from_numpy(rng.integers(-32, 33, (rows, k // 32, 32))).double() / 4
    # powers within the type's normal range
    p = torch.from_numpy(rng.integers(-10, 11, (rows, k // 32, 1))).double()
    ties = (mag * 2 ** p).to(dtype)
    smooth = (torch.from_numpy(rng.standard_normal((rows, k // 32, 32))) * 2 ** p).to(dtype)
    blocks[kind == 1] = 0.0
    blocks[kind == 2] = ties[kind == 2]
    blocks[kind > 3] = smooth[kind > 3]
    want_c, want_s = oq.mxfp4_quantize(x.double().numpy())
    got = gemm.quantize_rows_mxfp4(x.to(DEV))
    val = gemm.dequantize_rows_mxfp4(got)
    torch.cuda.synchronize()
    codes = torch.stack((got.codes & 15, got.codes >> 4), -1).view(rows, k).cpu().numpy()
    np.testing.assert_array_equal(gemm.mxfp4_block_scales(got.scales, rows, k).cpu().numpy(), want_s)
    np.testing.assert_array_equal(codes, want_c)
    want = torch.from_numpy(oq.mxfp4_dequantize(want_c, want_s)).bfloat16()  # exact: E2M1 has one mantissa bit
    assert torch.equal(val.cpu().view(torch.int16), want.view(torch.int16)) or (
        torch.equal(torch.isnan(val.cpu()), torch.isnan(want))
        and torch.equal(torch.nan_to_num(val.cpu()), torch.nan_to_num(want)))


@pytest.mark.parametrize("exponent", [-126, -100, -3, 0, 60, 125])
def test_quantiser_over_all_bf16_magnitudes(exponent):
    """Every positive finite bf16 value below 2^(exponent + 3) beside a block
    maximum that fixes X = exponent, both signs."""
    from ltx_amd.kernels import gemm

    bits = torch.arange(0, 0x7f80, dtype=torch.int16).view(torch.bfloat16)
    top = 2.0 ** (exponent + 2)
    v = bits[bits.double() < 2 * top]
    v = torch.cat((v, -v))
    v = torch.nn.functional.pad(v, (0, -v.numel() % 31)).view(-1, 31)
    x = torch.cat((torch.full((v.shape[0], 1), top, dtype=torch.bfloat16), v), 1)
    rows = x.shape[0]
    want_c, want_s = oq.mxfp4_quantize(x.double().numpy())
    assert (want_s == exponent + 127).all()
    got = gemm.quantize_rows_mxfp4(x.to(DEV))
    torch.cuda.synchronize()
    codes = torch.stack((got.codes & 15, got.codes >> 4), -1).view(rows, 32).cpu().numpy()
    np.testing.assert_array_equal(gemm.mxfp4_block_scales(got.scales, rows, 32).cpu().numpy(), want_s)
    np.testing.assert_array_equal(codes, want_c)


def test_quantiser_strided_rows_and_empty():
    from ltx_amd.kernels import gemm

    buf = torch.randn(37, 256, device=DEV).bfloat16()
    x = buf[:, 64:224]
    a, b = gemm.quantize_rows_mxfp4(x), gemm.quantize_rows_mxfp4(x.contiguous())
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales[:, :37], b.scales[:, :37])
    assert gemm.quantize_rows_mxfp4(x.view(37, 160)[:0]).shape == (0, 160)
    assert gemm.dequantize_rows_mxfp4(gemm.quantize_rows_mxfp4(x[:0])).shape == (0, 160)
    w = gemm.make_weight(torch.randn(64, 128, device=DEV).bfloat16(), kind="mxfp4")
    assert gemm.linear(torch.empty(0, 128, dtype=torch.bfloat16, device=DEV), w).shape == (0, 64)
    assert gemm.linear(torch.ones(2, 3, 128, dtype=torch.bfloat16, device=DEV), w).shape == (2, 3, 64)


def test_every_weight_scale_byte():
    """Columns with each E8M0 byte, against float64 (254: 2^127, 0: 2^-127)."""
    from ltx_amd.kernels import gemm

    n, k, m = 256, 128, 3
    codes = np.full((n, k), 2, np.uint8)  # 1.0
    scales = np.tile(np.arange(256, dtype=np.uint8)[:, None], (1, 4))
    b, w = oq.mxfp4_pack(codes, scales)
    x = torch.zeros(m, k, dtype=torch.bfloat16)
    x[0, 3], x[1, 64], x[2, 127] = 1.0, 2.0 ** -100, 2.0 ** 100
    wt = gemm.LinearWeight("mxfp4", torch.from_numpy(b).to(DEV), torch.from_numpy(w).to(DEV))
    got = gemm.linear(x.to(DEV), wt).double().cpu()
    want = (x.double() @ torch.from_numpy(oq.mxfp4_dequantize(codes, scales)).T)[:, :255]
    want = want.float().bfloat16().double()
    assert torch.isnan(got[:, 255]).all()
    # the matrix pipe may flush subnormals of the inputs and of the sum
    tiny = want.abs() < 2.0 ** -126
    sub = torch.arange(255) == 0
    ok = (got[:, :255] == want) | (tiny & (got[:, :255].abs() <= want.abs())) | (sub & (got[:, :255] == 0))
    assert ok.all(), (got[:, :255][~ok], want[~ok])


def test_streams_and_graphs():
    """A side stream; two captured graphs whose workspaces live at once,
    replayed alternately with eager work between, against the eager results."""
    from ltx_amd.kernels import gemm

    g = torch.Generator(device=DEV).manual_seed(1)
    cases = []
    for m, k, n in ((1, 4096, 4096), (68, 8192, 2048)):
        wt = gemm.make_weight((torch.randn(n, k, generator=g, device=DEV) * 0.02).bfloat16(),
                              torch.randn(n, generator=g, device=DEV), kind="mxfp4")
        x = torch.randn(m, k, generator=g, device=DEV).bfloat16()
        cases.append((x, wt))

    def work(x, wt):
        return gemm.linear(x, wt), gemm.linear(gemm.quantize_rows_mxfp4(x), wt)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = [work(*c) for c in cases]
    torch.cuda.current_stream().wait_stream(side)
    eager = [work(*c) for c in cases]
    torch.cuda.synchronize()
    for a, b in zip(there, eager):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    graphs, outs = [], []
    for c in cases:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(work(*c))
        graphs.append(gr)
    for it in range(3):
        for (x, _) in cases:
            x.copy_(torch.randn(x.shape, generator=g, device=DEV).bfloat16())
        want = [work(*c) for c in cases]
        for gr in graphs if it % 2 else graphs[::-1]:
            gr.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_rows_whose_strides_say_nothing():
    """One row under any stride, one row broadcast over many, a vector, one scale
    word row, a batch of rows."""
    from ltx_amd.kernels import gemm

    g = torch.Generator(device=DEV).manual_seed(4)
    col = torch.randn(128, 1, generator=g, device=DEV).bfloat16()
    w = gemm.make_weight(torch.randn(64, 128, generator=g, device=DEV).bfloat16(), kind="mxfp4")
    row = col.t()  # (1, 128), strides (1, 1)
    want = gemm.linear(row.contiguous(), w)
    assert torch.equal(gemm.linear(row, w), want)
    assert torch.equal(gemm.linear(row.expand(5, 128), w), want.expand(5, 64))
    assert torch.equal(gemm.linear(col[:, 0], w), want[0])
    a, b = gemm.quantize_rows_mxfp4(row), gemm.quantize_rows_mxfp4(row.contiguous())
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales[:, :1], b.scales[:, :1])
    e = gemm.quantize_rows_mxfp4(row.expand(5, 128))
    assert torch.equal(e.codes, b.codes.expand(5, 64)) and torch.equal(e.scales[:, :5], b.scales[:, :1].expand(1, 5))
    many = gemm.linear(e, w)
    assert torch.equal(many, gemm.linear(b, w).expand(5, 64))
    out = torch.empty(64, 1, dtype=torch.bfloat16, device=DEV).t()
    assert torch.equal(gemm.linear(row, w, out=out), want)
    with pytest.raises(ValueError):
        gemm.linear(row.expand(5, 128), w, out=out.expand(5, 64))
    res = torch.randn(64, 1, generator=g, device=DEV).bfloat16().t()
    gate = torch.randn(64, generator=g, device=DEV)
    kw = dict(epilogue=gemm.EPI_RESIDUAL, gate=gate)
    assert torch.equal(gemm.linear(row, w, residual=res, **kw), gemm.linear(row.contiguous(), w,
                                                                             residual=res.contiguous(), **kw))
    with pytest.raises(ValueError):
        gemm.linear(row.expand(5, 128), w, residual=res.expand(5, 64), **kw)


@pytest.mark.parametrize("m", [5, 200, 2200])
def test_misaligned_operands_are_refused(m):
    from ltx_amd import _lib
    from ltx_amd.kernels import gemm

    w = gemm.make_weight(torch.randn(64, 128, device=DEV).bfloat16(), kind="mxfp4")
    buf = torch.zeros(m, 160, dtype=torch.bfloat16, device=DEV)
    for x in (buf[:, 4:132], torch.zeros(m, 130, dtype=torch.bfloat16, device=DEV)[:, :128]):
        with pytest.raises(_lib.LtxKernelError):
            gemm.linear(x, w)
        with pytest.raises(_lib.LtxKernelError):
            gemm.quantize_rows_mxfp4(x)
    with pytest.raises(_lib.LtxKernelError):
        gemm.linear(buf[:, :128], w, out=torch.empty(m, 68, dtype=torch.bfloat16, device=DEV)[:, 4:])
    with pytest.raises(_lib.LtxKernelError):  # K of no 128: bf16 rows only
        v = gemm.make_weight(torch.randn(64, 192, device=DEV).bfloat16(), kind="mxfp4")
        gemm.linear(gemm.quantize_rows_mxfp4(torch.zeros(m, 192, device=DEV)), v)
    with pytest.raises(_lib.LtxKernelError):  # N of no 8
        v = gemm.make_weight(torch.randn(60, 128, device=DEV).bfloat16(), kind="mxfp4")
        gemm.linear(buf[:, :128], v)


@pytest.mark.parametrize("m", [1, 30, 50, 150, 900])
@pytest.mark.parametrize("k", [64, 192, 320, 1088])
def test_bytes_past_the_last_block_are_not_used(m, k):
    """Depths that end inside a scale word: its unused bytes may hold anything."""
    from ltx_amd.kernels import gemm

    n = 136
    wc, ws, w = _codes_words(n, k, seed=k)
    x = torch.randn(m, k, generator=torch.Generator(device=DEV).manual_seed(m), device=DEV).bfloat16()
    ws[-1] |= -65536  # blocks 2 and 3: NaN scales
    got = gemm.linear(x, gemm.LinearWeight("mxfp4", wc, ws))
    _check(got, *_reference(x.double(), w, None, "bias", None, None, None, False))
    val = gemm.dequantize(gemm.LinearWeight("mxfp4", wc, ws))
    assert torch.equal(val.double(), w)
