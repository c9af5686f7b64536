"""Rotary positions against float64.

A result a cos - b sin has two exact-in-fp32 inputs, a cosine and a sine that
are each within 2^-22 of the exact ones (the reduced turn is rounded to fp32,
2^-25 of a half turn at most: pi 2^-25 of an angle; sincospi is good to 2 ulp;
the factor's product rounds once), two fp32 roundings, and one rounding to the
type: |error| <= 2^-21 f (|a| + |b|) + half a step of the result.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _reference(x, positions, inv, layout, factor, transpose):
    d = 2 * inv.numel()
    t = positions.double()[..., None] * inv
    t = t[..., None, :]
    if t.dim() < x.dim():
        t = t[None]
    c, s = torch.cos(t) * factor, torch.sin(t) * factor * (-1 if transpose else 1)
    v = x.double()
    lo, hi = (slice(0, d // 2), slice(d // 2, d)) if layout == "half" else (slice(0, d, 2), slice(1, d, 2))
    a, b = v[..., lo], v[..., hi]
    out, err = v.clone(), torch.zeros_like(v)
    out[..., lo], out[..., hi] = a * c - b * s, b * c + a * s
    e = 2.0 ** -21 * abs(factor) * (a.abs() + b.abs())
    err[..., lo] = err[..., hi] = e
    step = torch.finfo(x.dtype).eps / 2
    rot = err > 0
    # half a step of the result; below the normal range, half its spacing
    spacing = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps / 2
    return out, err + torch.where(rot, step * (out.abs() + err) + spacing, torch.zeros_like(err))


def _check(got, x, *args):
    ref, err = _reference(x, *args)
    over = (got.double() - ref).abs() - err
    assert got.shape == x.shape and got.dtype == x.dtype
    assert over.max().item() <= 0, over.max().item()


@pytest.mark.parametrize("transpose", [False, True], ids=["fwd", "grad"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("tokens,heads,kv,dh,rot", [
    (1, 32, 32, 128, 128), (1, 1, 1, 2, 2), (3, 4, 2, 64, 32), (5, 3, 1, 80, 20), (7, 2, 2, 65, 64), (9, 5, 5, 66, 6),
    (64, 12, 4, 96, 96), (2100, 4, 1, 64, 16), (4099, 8, 8, 128, 64), (33, 2, 1, 512, 512), (130, 40, 3, 48, 46)])
def test_rotation(tokens, heads, kv, dh, rot, dtype, layout, transpose):
    from ltx_amd.kernels import rope_ops

    print(f"rotary T={tokens} H={heads}/{kv} dh={dh} rot={rot} {dtype} {layout} {transpose}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(tokens + dh)
    q = torch.randn(tokens, heads, dh, generator=g, device=DEV).to(dtype)
    k = torch.randn(tokens, kv, dh, generator=g, device=DEV).to(dtype)
    inv, _ = rope_ops.rotary_frequencies(rot)
    pos = torch.randint(0, 1 << 21, (tokens,), generator=g, device=DEV, dtype=torch.int32)
    oq, ok = rope_ops.rotary(q, k, pos, inv, layout=layout, factor=1.25, transpose=transpose)
    torch.cuda.synchronize()
    _check(oq, q, pos, inv, layout, 1.25, transpose)
    _check(ok, k, pos, inv, layout, 1.25, transpose)
    if rot < dh:
        assert torch.equal(oq[..., rot:], q[..., rot:]) and torch.equal(ok[..., rot:], k[..., rot:])
    iq, ik = q.clone(), k.clone()
    rope_ops.rotary(iq, ik, pos, inv, layout=layout, factor=1.25, transpose=transpose, out=(iq, ik))
    assert torch.equal(iq, oq) and torch.equal(ik, ok)


@pytest.mark.parametrize("pdtype", [torch.int32, torch.int64, torch.float32, torch.float64], ids=str)
@pytest.mark.parametrize("own_rows", [False, True])
def test_batches_strides_and_position_types(pdtype, own_rows):
    """(B, T) batches in (B, T, H, dh) and transposed (B, H, T, dh) storage, odd
    offsets, queries and keys inside one fused projection, k absent."""
    from ltx_amd.kernels import rope_ops

    b, t, h, dh = 3, 37, 4, 64
    g = torch.Generator(device=DEV).manual_seed(3)
    inv, f = rope_ops.rotary_frequencies(32, scaling="yarn", stretch=16)
    pos = torch.randint(0, 5000, (b, t) if own_rows else (t,), generator=g, device=DEV).to(pdtype)
    if pdtype.is_floating_point:
        pos = pos + 0.375
    fused = torch.randn(b, t, 3 * h * dh, generator=g, device=DEV).bfloat16()
    q = fused[..., :h * dh].unflatten(-1, (h, dh))
    k = fused[..., h * dh:2 * h * dh].unflatten(-1, (h, dh))
    for layout in rope_ops.ROTARY_LAYOUTS:
        oq, ok = rope_ops.rotary(q, k, pos, inv, layout=layout, factor=f)
        _check(oq, q, pos, inv, layout, f, False)
        _check(ok, k, pos, inv, layout, f, False)
        hq = torch.randn(b, h, t, dh, generator=g, device=DEV).transpose(1, 2)
        out = torch.full((b, t + 1, h, dh + 3), 9.0, device=DEV)
        o, none = rope_ops.rotary(hq, None, pos, inv, layout=layout, out=(out[:, 1:, :, 1:dh + 1], None))
        assert none is None
        _check(o, hq, pos, inv, layout, 1.0, False)
        rest = out.clone()
        rest[:, 1:, :, 1:dh + 1] = 9.0
        assert (rest == 9.0).all()
        # in place inside the projection: the values keep what they had
        copy = fused.clone()
        rope_ops.rotary(copy[..., :h * dh].unflatten(-1, (h, dh)), copy[..., h * dh:2 * h * dh].unflatten(-1, (h, dh)),
                        pos, inv, layout=layout, factor=f,
                        out=(copy[..., :h * dh].unflatten(-1, (h, dh)),
                             copy[..., h * dh:2 * h * dh].unflatten(-1, (h, dh))))
        assert torch.equal(copy[..., 2 * h * dh:], fused[..., 2 * h * dh:])
        assert torch.equal(copy[..., :h * dh].unflatten(-1, (h, dh)), oq)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient_is_the_transposed_rotation(layout):
    """<R x, g> against differences in x, and against autograd of the formula."""
    from ltx_amd.kernels import rope_ops

    g = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn(6, 2, 20, generator=g, device=DEV)
    up = torch.randn(6, 2, 20, generator=g, device=DEV)
    inv, _ = rope_ops.rotary_frequencies(12)
    pos = torch.arange(6, device=DEV) * 1000
    grad, _ = rope_ops.rotary(up, None, pos, inv, layout=layout, factor=1.5, transpose=True)
    leaf = x.double().requires_grad_()
    ref, _ = _reference(leaf, pos, inv, layout, 1.5, False)
    want, = torch.autograd.grad((ref * up.double()).sum(), leaf)
    # as a forward result: 2^-21 f (|a| + |b|) and half a step
    assert (grad.double() - want).abs().max() <= 2.0 ** -21 * 1.5 * 2 * up.abs().max() + 2.0 ** -24 * grad.abs().max()
    for i in ((0, 0, 0), (3, 1, 5), (5, 0, 11), (4, 1, 17)):
        h = 0.5  # the map is linear: no truncation error, only rounding of the two results
        d = torch.zeros_like(x)
        d[i] = h
        plus, _ = rope_ops.rotary(x + d, None, pos, inv, layout=layout, factor=1.5)
        minus, _ = rope_ops.rotary(x - d, None, pos, inv, layout=layout, factor=1.5)
        diff = ((plus.double() - minus.double()) * up.double()).sum() / (2 * h)
        assert abs(diff.item() - grad[i].item()) <= 2.0 ** -19 * 1.5 * (x.abs().max() + h).item() * up[i[0], i[1]].abs().sum().item()


def test_agrees_with_the_table_form():
    """The split RoPE of the QK-norm kernel's tables, from positions instead:
    norm weights of one and rows of unit mean square leave only the rotation."""
    from ltx_amd.kernels import rope_ops

    t, heads, dh = 40, 16, 64
    g = torch.Generator(device=DEV).manual_seed(6)
    x = (torch.randint(0, 2, (t, heads * dh), generator=g, device=DEV) * 2 - 1).bfloat16()  # +-1: mean square 1
    inv, _ = rope_ops.rotary_frequencies(dh)
    pos = torch.arange(t, device=DEV)
    ang = (pos.double()[:, None] * inv).repeat(1, heads)
    pe = (torch.cos(ang).float(), torch.sin(ang).float())
    q = x.clone()
    ones = torch.ones(heads * dh, device=DEV)
    rope_ops.qknorm_rope_(q, ones, pe, q[:0], ones, None, heads, eps=0.0)
    out, _ = rope_ops.rotary(x.view(t, heads, dh), None, pos, inv)
    torch.cuda.synchronize()
    # both within 2^-21 * 2 and half a bf16 step (2^-8) of the same value
    d = (q.view_as(out).double() - out.double()).abs()
    assert (d <= 2 * (2.0 ** -8 * out.double().abs() + 2.0 ** -20)).all()


def test_streams_graph_and_empty():
    from ltx_amd.kernels import rope_ops

    inv, _ = rope_ops.rotary_frequencies(64)
    q = torch.randn(50, 4, 64, device=DEV).bfloat16()
    pos = torch.arange(50, device=DEV, dtype=torch.int32)
    assert rope_ops.rotary(q[:0], None, pos[:0], inv)[0].shape == (0, 4, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, _ = rope_ops.rotary(q, None, pos, inv)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, rope_ops.rotary(q, None, pos, inv)[0])
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out, _ = rope_ops.rotary(q, None, pos, inv)
    for i in range(3):
        pos.add_(1000)
        q.copy_(torch.randn(50, 4, 64, device=DEV))
        want, _ = rope_ops.rotary(q, None, pos, inv)
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_quantised_projection_rotation_attention():
    """A run as an attention layer makes it: MXFP4 projection of queries, keys
    and values, rotation of the first two in place, attention, MXFP4 output
    projection -- against float64 of the decoded weights, with the bf16
    roundings between the operators applied to the reference as well."""
    from ltx_amd.kernels import attention, gemm, rope_ops

    t, heads, dh = 200, 8, 64
    inner = heads * dh
    g = torch.Generator(device=DEV).manual_seed(9)
    wqkv = gemm.make_weight((torch.randn(3 * inner, 1024, generator=g, device=DEV) / 32).bfloat16(),
                            torch.randn(3 * inner, generator=g, device=DEV) * 0.1, kind="mxfp4")
    wo = gemm.make_weight((torch.randn(1024, inner, generator=g, device=DEV) / 23).bfloat16(), kind="mxfp4")
    x = torch.randn(t, 1024, generator=g, device=DEV).bfloat16()
    inv, f = rope_ops.rotary_frequencies(dh, scaling="linear", stretch=4)
    pos = torch.arange(t, device=DEV)
    buf = gemm.linear(x, wqkv)
    q, k, v = buf.split(inner, 1)
    qh, kh = q.unflatten(1, (heads, dh)), k.unflatten(1, (heads, dh))
    rope_ops.rotary(qh, kh, pos, inv, layout="interleaved", factor=f, out=(qh, kh))
    o = attention.flash_attention(q, k, v, heads)
    y = gemm.linear(o, wo)
    torch.cuda.synchronize()

    ref = (x.double() @ gemm.dequantize(wqkv).double().T + wqkv.bias.double()).bfloat16()
    rq, rk, rv = (a.unflatten(1, (heads, dh)) for a in ref.split(inner, 1))
    rq = _reference(rq, pos, inv, "interleaved", f, False)[0].bfloat16().double()
    rk = _reference(rk, pos, inv, "interleaved", f, False)[0].bfloat16().double()
    p = torch.softmax(torch.einsum("qhd,khd->hqk", rq, rk) * dh ** -0.5, -1)
    ro = torch.einsum("hqk,khd->qhd", p, rv.double()).reshape(t, inner).bfloat16()
    want = ro.double() @ gemm.dequantize(wo).double().T
    # every operator is held to its own bound in its own test; here a rounding
    # step of an intermediate may fall the other way: 2^-8 relative per stage,
    # four stages, in the 2-norm
    assert (y.double() - want).norm() <= 4 * 2.0 ** -8 * want.norm()
