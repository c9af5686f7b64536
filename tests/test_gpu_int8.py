"""int8 rows and int8 x int8 products against float64.

Codes and scales are held to the rule bit for bit.  A product's sum is exact in
int32; its value is ((sum sa) sw) + bias in fp32: the sum's conversion, two
products and one sum, each off by 2^-24 of its result, so |error| <= 2^-22 (|p| +
|bias|) with p the scaled sum; what the epilogue makes of that, and half a bf16 step
(2^-8) of the result.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _rule(x):
    """The format's rule on the host: quotients of fp32 values rounded to fp32 (by way of fp64, which rounds a
    quotient of fp32 values to the same fp32 value)."""
    v = x.detach().cpu().double()
    bad = ~torch.isfinite(v).all(1)
    scale = (v.abs().amax(1) / 127).float()
    q = torch.round((v / scale.double()[:, None]).float()).clamp(-127, 127)
    q = torch.where((scale > 0)[:, None] & ~bad[:, None], q, torch.zeros_like(q))
    return q.to(torch.int8), torch.where(bad, torch.full_like(scale, math.nan), scale)


def _check_rows(x):
    from ltx_amd.kernels import gemm

    rows = gemm.quantize_rows_int8(x)
    torch.cuda.synchronize()
    q, s = _rule(x.reshape(-1, x.shape[-1]))
    assert torch.equal(rows.scales.cpu().nan_to_num(-1.0), s.nan_to_num(-1.0))
    assert torch.equal(rows.codes.cpu(), q), (rows.codes.cpu() != q).sum()
    back = gemm.dequantize_rows_int8(rows).cpu()
    want = (q.float() * s[:, None]).bfloat16()
    assert torch.equal(back.isnan(), want.isnan()) and torch.equal(back.nan_to_num(0.0), want.nan_to_num(0.0))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,k", [(1, 16), (1, 4096), (3, 48), (68, 2048), (5, 4112), (1030, 528), (2, 16384),
                                    (3, 16400), (4, 40000), (1500, 4096)])
def test_rows(rows, k, dtype):
    print(f"int8 rows {rows} x {k} {dtype}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(rows + k)
    x = torch.randn(rows, k, generator=g, device=DEV)
    x[:, ::7] *= 30
    _check_rows(x.to(dtype))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rows_at_the_borders(dtype):
    """Quotients at or next to a half, zeros, the type's extremes and subnormals, NaN and infinities."""
    top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    cases = []
    for amax in (127.0, 127.0 / 64, 254.0, 63.5, 101.0, 1.0, 0.7, top, tiny * 127, tiny * 3, tiny):
        a = torch.tensor(amax, dtype=torch.float64).to(dtype).double()
        steps = (torch.arange(-254, 255, dtype=torch.float64) / 2)
        v = (steps * a / 127).to(dtype)
        up = torch.nextafter(v.float(), torch.full_like(v.float(), math.inf)).to(dtype)
        v = torch.cat((v, up, -up, torch.full((5,), a.item(), dtype=torch.float64).to(dtype)))
        v = v[v.double().abs() <= a]
        cases.append(torch.cat((v, torch.zeros(1552 - len(v), dtype=dtype))))
    zero, nan, inf = (torch.zeros(1552, dtype=dtype) for _ in range(3))
    nan[7], inf[1551] = math.nan, -math.inf
    both = nan.clone()
    both[9], both[10] = math.inf, 3.0
    _check_rows(torch.stack(cases + [zero, nan, inf, both, -zero]).to(DEV))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rows_of_any_layout(dtype):
    g = torch.Generator(device=DEV).manual_seed(1)
    wide = torch.randn(6, 5, 96, generator=g, device=DEV).to(dtype)
    for x in (wide[..., :64], wide[..., 32:80], wide[:, 2, 16:], wide[3, 2], wide.transpose(0, 1), wide[0, :1].expand(9, 96),
              wide.flatten()[1:].as_strided((4, 32), (96, 1)).clone(), wide[::2, ::2]):
        _check_rows(x)


def _case(m, n, k, seed=0, bias=True):
    from ltx_amd.kernels import gemm

    g = torch.Generator(device=DEV).manual_seed(seed + m + n + k)
    codes = torch.randint(-127, 128, (m, k), generator=g, device=DEV, dtype=torch.int8)
    xs = torch.rand(m, generator=g, device=DEV) * 0.02 + 0.001
    w = torch.randint(-127, 128, (n, k), generator=g, device=DEV, dtype=torch.int8)
    ws = (torch.rand(n, generator=g, device=DEV) * 0.02 + 0.001) / math.sqrt(k)
    b = torch.randn(n, generator=g, device=DEV) if bias else None
    return gemm.Int8Rows(codes, xs), gemm.LinearWeight("int8", w, ws, b)


def _scaled(rows, weight):
    return (rows.codes.double() @ weight.w.double().T) * rows.scales.double()[:, None] * weight.scale.double()


def _epilogue(p, weight, epilogue, residual, gate, sigmoid_from):
    """Result and bound in float64 from the scaled sums."""
    b = 0.0 if weight.bias is None else weight.bias.double()
    y = p + b
    e = 2.0 ** -22 * (p.abs() + torch.as_tensor(b, device=p.device).abs())
    if weight.qlinear and weight.bias is not None:
        e = e + 2.0 ** -8 * p.abs()
    half = 2.0 ** -8
    # hardware exp2 and reciprocal: 2^-22 each, an exponent of at most 2^7 rounded to 2^-23 of itself
    soft = 2.0 ** -15
    if epilogue == 1:
        ref = torch.nn.functional.gelu(y, approximate="tanh")
        return ref, (half + soft) * ref.abs() + 1.2 * e + 1e-30
    if epilogue == 4:
        ref = 2 * torch.sigmoid(y)
        return ref, (half + soft) * ref + e
    if epilogue in (2, 3):
        ref = residual.double() + gate.double() * y
        err = gate.double().abs() * e + half * ref.abs() * (1 + 2.0 ** -8)
        if epilogue == 3:  # the branch and its product are rounded too
            err = err + 2.02 * half * (gate.double() * y).abs() * (1 + half)
        return ref, err + 2.0 ** -23 * ref.abs()
    if sigmoid_from is not None:
        ref = torch.cat((y[:, :sigmoid_from], 2 * torch.sigmoid(y[:, sigmoid_from:])), 1)
        return ref, (half + soft) * ref.abs() + e
    return y, half * y.abs() + e


SHAPES = [(1, 8, 64), (1, 4096, 4096), (2, 264, 192), (16, 128, 1088), (17, 72, 64), (33, 520, 448), (64, 2048, 2048),
          (68, 2048, 8192), (96, 136, 320), (130, 264, 576), (257, 1032, 704), (300, 4096, 1024), (1296, 2056, 512),
          (520, 8192, 256), (2049, 520, 1216), (3456, 1040, 320)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_products(m, n, k):
    from ltx_amd.kernels import gemm

    print(f"int8 product {m} x {k} -> {n}", flush=True)
    rows, weight = _case(m, n, k)
    p = _scaled(rows, weight)
    g = torch.Generator(device=DEV).manual_seed(2)
    residual = torch.randn(m, n, generator=g, device=DEV).bfloat16()
    gate = torch.randn(n, generator=g, device=DEV)
    for epilogue, sig in ((0, None), (0, n - 8), (0, max(n - 40, 0)), (1, None), (2, None), (3, None), (4, None)):
        kw = dict(residual=residual, gate=gate) if epilogue in (2, 3) else {}
        y = gemm.linear(rows, weight, epilogue=epilogue, sigmoid_from=sig, **kw)
        torch.cuda.synchronize()
        ref, err = _epilogue(p, weight, epilogue, residual, gate, sig)
        over = ((y.double() - ref).abs() - err).max().item()
        assert y.shape == (m, n) and y.dtype is torch.bfloat16 and over <= 0, (epilogue, sig, over)


@pytest.mark.parametrize("m,n,k", [(520, 24576, 192), (1299, 12328, 576), (4100, 4104, 448), (1025, 4096, 16384),
                                   (1500, 12744, 320)])
def test_products_of_a_round_of_tall_tiles(m, n, k):
    """Sizes that one round of the tallest tiles takes, a part of them in K ranges; and whole rounds with rows left over."""
    test_products(m, n, k)


@pytest.mark.parametrize("m", [1, 40, 300, 2100])
def test_largest_sums_are_exact(m):
    """Codes of +-127 and -128 at the largest depth: sums near 2^31, whose fp32 value rounds once."""
    from ltx_amd.kernels import gemm

    k, n = 131008, 16
    codes = torch.full((m, k), -128, dtype=torch.int8, device=DEV)
    w = torch.full((n, k), -128, dtype=torch.int8, device=DEV)
    w[1], w[2, ::2], w[3, 5:] = 127, 127, 0
    one = torch.ones(m, device=DEV), torch.full((n,), 2.0 ** -31, device=DEV)
    weight = gemm.LinearWeight("int8", w, one[1])
    y = gemm.linear(gemm.Int8Rows(codes, one[0]), weight)
    want = (w.long() * -128).sum(1).double() * 2.0 ** -31
    assert ((y.double() - want).abs() <= 2.0 ** -8 * want.abs()).all()


@pytest.mark.parametrize("n,k", [(264, 640), (2048, 1024), (4104, 4096)])
def test_rows_give_the_same_bits_in_every_product(n, k):
    """However many rows share a call, and whatever kernel and K ranges it takes."""
    from ltx_amd.kernels import gemm

    rows, weight = _case(2600, n, k, seed=5)
    g = torch.Generator(device=DEV).manual_seed(6)
    residual = torch.randn(2600, n, generator=g, device=DEV).bfloat16()
    gate = torch.randn(n, generator=g, device=DEV)

    for epilogue in (0, 1, 2, 3, 4):
        def part(a, b):
            kw = dict(residual=residual[a:b], gate=gate) if epilogue in (2, 3) else {}
            return gemm.linear(gemm.Int8Rows(rows.codes[a:b], rows.scales[a:b]), weight, epilogue=epilogue, **kw)

        whole = part(0, 2600)
        for a, b in ((0, 1), (7, 23), (100, 132), (640, 708), (1000, 1128), (3, 203), (2000, 2600), (500, 1900)):
            assert torch.equal(part(a, b), whole[a:b]), (epilogue, a, b)


def test_strides_outputs_and_absent_bias():
    from ltx_amd.kernels import gemm

    for m, n, k in ((1, 64, 128), (9, 264, 192), (200, 264, 192), (700, 1024, 512)):
        rows, weight = _case(m, n, k, bias=False)
        wide = torch.zeros(m, k + 32, dtype=torch.int8, device=DEV)
        wide[:, 16:k + 16] = rows.codes
        ww = torch.zeros(n, k + 48, dtype=torch.int8, device=DEV)
        ww[:, 32:k + 32] = weight.w
        want = gemm.linear(rows, weight)
        buf = torch.full((m + 2, n + 24), 7.0, device=DEV).bfloat16()
        out = buf[1:m + 1, 8:n + 8]
        got = gemm.linear(gemm.Int8Rows(wide[:, 16:k + 16], rows.scales),
                          gemm.LinearWeight("int8", ww[:, 32:k + 32], weight.scale), out=out)
        assert got is out and torch.equal(got, want)
        out.fill_(7.0)
        assert (buf == 7.0).all()  # nothing beside it was written
        # scales at odd addresses, the residual updated in place
        odd = torch.zeros(m + n + 1, device=DEV)
        odd[1:m + 1], odd[m + 1:] = rows.scales, weight.scale
        res = torch.randn(m, n, device=DEV).bfloat16()
        gate = torch.randn(n, device=DEV)
        kw = dict(epilogue=gemm.EPI_RESIDUAL, gate=gate)
        fresh = gemm.linear(rows, weight, residual=res, **kw)
        gemm.linear(gemm.Int8Rows(rows.codes, odd[1:m + 1]), gemm.LinearWeight("int8", weight.w, odd[m + 1:]), residual=res,
                    out=res, **kw)
        assert torch.equal(res, fresh)
        q = gemm.LinearWeight("int8", weight.w, weight.scale, torch.randn(n, device=DEV), qlinear=True)
        ref, err = _epilogue(_scaled(rows, q), q, 0, None, None, None)
        assert ((gemm.linear(rows, q).double() - ref).abs() <= err).all()


def test_rows_of_zeros_and_of_nan():
    """A NaN or an infinity in a row makes that row NaN and leaves the others."""
    from ltx_amd.kernels import gemm

    for m in (3, 70, 600):
        x = torch.randn(m, 256, device=DEV)
        x[1], x[2, 9] = 0, math.inf
        x[m - 1, 255] = math.nan
        _, weight = _case(1, 136, 256)
        y = gemm.linear(gemm.quantize_rows_int8(x), weight)
        assert torch.equal(y[1], weight.bias.bfloat16())
        bad = [2, m - 1]
        assert y[bad].isnan().all() and not y[[i for i in range(m) if i not in bad]].isnan().any()


def test_far_rows():
    """Operand rows past 2^31 bytes, outputs past 2^32."""
    from ltx_amd.kernels import gemm

    m, n, k = 33000, 72, 320
    rows, weight = _case(m, n, k)
    far = torch.empty(m, 1 << 17, dtype=torch.int8, device=DEV)[:, 64:64 + k]
    far.copy_(rows.codes)
    out = torch.empty(m, 1 << 16, dtype=torch.bfloat16, device=DEV)[:, 8:8 + n]
    got = gemm.linear(gemm.Int8Rows(far, rows.scales), weight, out=out)
    assert torch.equal(got, gemm.linear(rows, weight))
    x = torch.empty(m, 1 << 16, dtype=torch.bfloat16, device=DEV)[:, 64:64 + k]
    x.copy_(torch.randn(m, k, device=DEV))
    a, b = gemm.quantize_rows_int8(x), gemm.quantize_rows_int8(x.contiguous())
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


def test_empty():
    from ltx_amd.kernels import gemm

    _, weight = _case(1, 64, 128)
    rows = gemm.quantize_rows_int8(torch.zeros(0, 128, device=DEV))
    assert rows.codes.shape == (0, 128) and rows.scales.shape == (0,)
    assert gemm.dequantize_rows_int8(rows).shape == (0, 128) and gemm.linear(rows, weight).shape == (0, 64)


@pytest.mark.parametrize("m", [1, 68, 600])
def test_streams_and_graphs(m):
    """Two streams at once, and two captured products replayed with eager work between."""
    from ltx_amd.kernels import gemm

    _, wa = _case(1, 2048, 4096, seed=1)
    _, wb = _case(1, 1032, 2048, seed=2)
    x = torch.randn(m, 4096, device=DEV).bfloat16()

    def both(v):
        h = gemm.linear(gemm.quantize_rows_int8(v), wa, epilogue=gemm.EPI_GELU)
        return gemm.linear(gemm.quantize_rows_int8(h), wb)

    want = both(x)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got += [both(x) for _ in range(4)]
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(x)
    for _ in range(3):
        x.copy_(torch.randn(m, 4096, device=DEV))
        want = both(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
