"""The per-head norm with rotary positions, and its gradient, against float64.

A sum over a head's channels adds at most 40 fp32 values one after another (16
channels of a lane, six exchanges; 32 and six where a head has more than 64 items):
2^-18.6 of a sum of positive terms, half of that in its root; with the mean, eps, the
root and the products around it at most 2^-19 of r x u.  Rotation: 2^-21 f (|a| + |b|)
(test_gpu_rotary.py).  So |error| <= 2^-18 f (|a| + |b|) and half a step of the
result's type.  The gradient's bound follows its formula with the same terms.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
EPS = 1e-5


def _halves(d, layout):
    return (slice(0, d // 2), slice(d // 2, d)) if layout == "half" else (slice(0, d, 2), slice(1, d, 2))


def _turn(v, positions, inv, layout, factor, back=False):
    """(rotated values, |a| + |b| times the factor) in float64."""
    if inv is None:
        return v, v.abs()
    t = (positions.double()[..., None] * inv)[..., None, :]
    if t.dim() < v.dim():
        t = t[None]
    c, s = torch.cos(t) * factor, torch.sin(t) * factor * (-1 if back else 1)
    lo, hi = _halves(2 * inv.numel(), layout)
    a, b = v[..., lo], v[..., hi]
    out, size = v.clone(), v.abs().clone()
    out[..., lo], out[..., hi] = a * c - b * s, b * c + a * s
    size[..., lo] = size[..., hi] = abs(factor) * (a.abs() + b.abs())
    return out, size


def _step(ref, err, dtype):
    f = torch.finfo(dtype)
    return f.eps / 2 * (ref.abs() + err) + f.smallest_normal * f.eps / 2


def _forward(x, w, positions, inv, layout="half", factor=1.0, offset=0.0, eps=EPS):
    v = x.double()
    z = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps)
    if w is not None:
        z = z * (offset + w.double())
    y, size = _turn(z, positions, inv, layout, factor)
    err = 2.0 ** -18 * size
    return y, err + _step(y, err, x.dtype)


def _gradient(g, x, w, positions, inv, layout="half", factor=1.0, offset=0.0, eps=EPS):
    """((dx, bound), (dw, bound) or None)"""
    v, up = x.double(), g.double()
    r = torch.rsqrt(v.square().mean(-1, keepdim=True) + eps)
    n = v * r
    gz, size = _turn(up, positions, inv, layout, factor, back=True)
    ez = 2.0 ** -21 * size
    u = torch.ones((), dtype=torch.float64, device=x.device) if w is None else offset + w.double()
    gn = gz * u
    k = (gn * n).mean(-1, keepdim=True)
    # the sum of k: its terms' errors, 40 additions, and r's 2^-19
    ek = (u.abs() * ez * n.abs()).mean(-1, keepdim=True) + 2.0 ** -18 * (gn * n).abs().mean(-1, keepdim=True)
    dx = r * (gn - n * k)
    err = r * (u.abs() * ez + n.abs() * ek) + 2.0 ** -18 * r * (gn.abs() + (n * k).abs())
    out = (dx, err + _step(dx, err, x.dtype))
    if w is None:
        return out, None
    over = tuple(range(x.dim() - 1))
    # terms gz n, of which a lane adds at most 512 one after another at these sizes
    term = (gz * n).abs()
    return out, ((gz * n).sum(over), (ez * n.abs()).sum(over) + (2.0 ** -18 + 2.0 ** -15) * term.sum(over) + 1e-30)


def _within(got, want):
    ref, err = want
    assert got.shape == ref.shape
    over = ((got.double() - ref).abs() - err).max().item() if got.numel() else 0.0
    assert over <= 0, over


def _inputs(tokens, heads, kv, dh, rot, dtype, weights=True, seed=0):
    from ltx_amd.kernels import rope_ops

    g = torch.Generator(device=DEV).manual_seed(seed + tokens + dh)
    q, k, gq, gk = (torch.randn(tokens, h, dh, generator=g, device=DEV).mul(s).to(dtype)
                    for h, s in ((heads, 3.0), (kv, 0.2), (heads, 1.0), (kv, 1.0)))
    wq, wk = (torch.randn(dh, generator=g, device=DEV) * 0.3 + 1 for _ in range(2)) if weights else (None, None)
    inv = rope_ops.rotary_frequencies(rot)[0] if rot else None
    pos = torch.randint(0, 1 << 21, (tokens,), generator=g, device=DEV, dtype=torch.int32) if rot else None
    return q, k, gq, gk, wq, wk, pos, inv


SHAPES = [(1, 32, 8, 128, 128), (1, 1, 1, 2, 2), (3, 4, 2, 64, 32), (5, 3, 1, 80, 20), (7, 2, 2, 65, 64),
          (9, 5, 5, 66, 6), (64, 12, 4, 96, 96), (2100, 4, 1, 64, 16), (4099, 8, 8, 128, 64), (33, 2, 1, 512, 512),
          (130, 40, 3, 48, 46), (6, 3, 2, 511, 510), (11, 2, 1, 512, 2), (17, 3, 1, 1, 0), (40, 6, 2, 127, 0),
          (50, 4, 4, 128, 0), (21, 2, 2, 512, 120), (1300, 1, 1, 256, 256)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("tokens,heads,kv,dh,rot", SHAPES)
def test_forward_and_gradient(tokens, heads, kv, dh, rot, dtype, layout):
    from ltx_amd.kernels import rope_ops

    print(f"headnorm T={tokens} H={heads}/{kv} dh={dh} rot={rot} {dtype} {layout}", flush=True)
    q, k, gq, gk, wq, wk, pos, inv = _inputs(tokens, heads, kv, dh, rot, dtype)
    how = dict(layout=layout, factor=1.25 if rot else 1.0)
    for offset in (0.0, 1.0):
        oq, ok = rope_ops.headnorm_rotary(q, k, wq, wk, pos, inv, eps=EPS, weight_offset=offset, **how)
        torch.cuda.synchronize()
        assert oq.dtype is dtype
        _within(oq, _forward(q, wq, pos, inv, offset=offset, **how))
        _within(ok, _forward(k, wk, pos, inv, offset=offset, **how))
        dq, dk, dwq, dwk = rope_ops.headnorm_rotary_grad(gq, gk, q, k, wq, wk, pos, inv, eps=EPS, weight_offset=offset,
                                                         **how)
        torch.cuda.synchronize()
        assert dq.dtype is dtype and dwq.dtype is torch.float32
        for got, dw, args in ((dq, dwq, (gq, q, wq)), (dk, dwk, (gk, k, wk))):
            want, sums = _gradient(*args, pos, inv, offset=offset, **how)
            _within(got, want)
            _within(dw, sums)
    # the same bits in place and again
    iq, ik = q.clone(), k.clone()
    rope_ops.headnorm_rotary(iq, ik, wq, wk, pos, inv, eps=EPS, weight_offset=1.0, out=(iq, ik), **how)
    assert torch.equal(iq, oq) and torch.equal(ik, ok)
    for into in ((q.clone(), k.clone()), (gq.clone(), gk.clone())):
        a = dict(gq=gq, gk=gk, q=q, k=k)
        a.update(zip(("q", "k") if torch.equal(into[0], q) else ("gq", "gk"), into))
        again = rope_ops.headnorm_rotary_grad(a["gq"], a["gk"], a["q"], a["k"], wq, wk, pos, inv, eps=EPS,
                                              weight_offset=1.0, out=into, **how)
        assert again[0] is into[0] and all(torch.equal(x, y) for x, y in zip(again, (dq, dk, dwq, dwk)))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_without_weights_keys_or_one_of_them(dtype):
    from ltx_amd.kernels import rope_ops

    q, k, gq, gk, wq, wk, pos, inv = _inputs(37, 4, 2, 64, 32, dtype)
    for a, b in ((None, None), (wq, None), (None, wk)):
        oq, ok = rope_ops.headnorm_rotary(q, k, a, b, pos, inv, eps=EPS)
        _within(oq, _forward(q, a, pos, inv))
        _within(ok, _forward(k, b, pos, inv))
        dq, dk, da, db = rope_ops.headnorm_rotary_grad(gq, gk, q, k, a, b, pos, inv, eps=EPS)
        for got, dw, args in ((dq, da, (gq, q, a)), (dk, db, (gk, k, b))):
            want, sums = _gradient(*args, pos, inv)
            _within(got, want)
            assert (dw is None) == (sums is None)
            if dw is not None:
                _within(dw, sums)
    oq, none = rope_ops.headnorm_rotary(q, None, wq, None, pos, inv, eps=EPS)
    assert none is None
    _within(oq, _forward(q, wq, pos, inv))
    dq, none, dw, no_weight = rope_ops.headnorm_rotary_grad(gq, None, q, None, wq, None, pos, inv, eps=EPS)
    assert none is None and no_weight is None
    _within(dq, _gradient(gq, q, wq, pos, inv)[0])
    _within(dw, _gradient(gq, q, wq, pos, inv)[1])


@pytest.mark.parametrize("pdtype", [torch.int32, torch.int64, torch.float32, torch.float64], ids=str)
@pytest.mark.parametrize("own_rows", [False, True])
def test_batches_strides_and_position_types(pdtype, own_rows):
    """(B, T) batches inside a fused projection, in transposed storage, at odd offsets, gradients that are one value
    for all tokens."""
    from ltx_amd.kernels import rope_ops

    b, t, h, dh = 3, 37, 4, 64
    g = torch.Generator(device=DEV).manual_seed(3)
    inv, f = rope_ops.rotary_frequencies(32, scaling="yarn", stretch=16)
    pos = torch.randint(0, 5000, (b, t) if own_rows else (t,), generator=g, device=DEV).to(pdtype)
    if pdtype.is_floating_point:
        pos = pos + 0.375
    wq, wk = (torch.randn(dh, generator=g, device=DEV) for _ in range(2))
    fused = torch.randn(b, t, 3 * h * dh, generator=g, device=DEV).bfloat16()
    q, k = (fused[..., i * h * dh:(i + 1) * h * dh].unflatten(-1, (h, dh)) for i in range(2))
    for layout in rope_ops.ROTARY_LAYOUTS:
        how = dict(layout=layout, factor=f)
        oq, ok = rope_ops.headnorm_rotary(q, k, wq, wk, pos, inv, eps=EPS, **how)
        _within(oq, _forward(q, wq, pos, inv, **how))
        _within(ok, _forward(k, wk, pos, inv, **how))
        hq = torch.randn(b, h, t, dh, generator=g, device=DEV).transpose(1, 2)
        out = torch.full((b, t + 1, h, dh + 3), 9.0, device=DEV)
        o, _ = rope_ops.headnorm_rotary(hq, None, wq, None, pos, inv, eps=EPS, out=(out[:, 1:, :, 1:dh + 1], None), **how)
        _within(o, _forward(hq, wq, pos, inv, **how))
        rest = out.clone()
        rest[:, 1:, :, 1:dh + 1] = 9.0
        assert (rest == 9.0).all()
        copy = fused.clone()
        views = tuple(copy[..., i * h * dh:(i + 1) * h * dh].unflatten(-1, (h, dh)) for i in range(2))
        rope_ops.headnorm_rotary(*views, wq, wk, pos, inv, eps=EPS, out=views, **how)
        assert torch.equal(copy[..., 2 * h * dh:], fused[..., 2 * h * dh:])
        assert torch.equal(views[0], oq) and torch.equal(views[1], ok)
        up = torch.randn(b, 1, h, dh, generator=g, device=DEV).expand(b, t, h, dh)
        dq, _, dw, _ = rope_ops.headnorm_rotary_grad(up, None, hq, None, wq, None, pos, inv, eps=EPS,
                                                     out=(out[:, :-1, :, 2:dh + 2], None), **how)
        want, sums = _gradient(up, hq, wq, pos, inv, **how)
        _within(dq, want)
        _within(dw, sums)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient_against_autograd_and_differences(layout):
    from ltx_amd.kernels import rope_ops

    q, _, gq, _, w, _, pos, inv = _inputs(6, 3, 1, 20, 12, torch.float32)
    how = dict(layout=layout, factor=1.5, offset=1.0)
    dq, _, dw, _ = rope_ops.headnorm_rotary_grad(gq, None, q, None, w, None, pos, inv, eps=EPS, weight_offset=1.0,
                                                 layout=layout, factor=1.5)

    def loss(x, v):
        return (_forward(x, v, pos, inv, **how)[0] * gq.double()).sum()

    leaf, wl = q.double().requires_grad_(), w.double().requires_grad_()
    want = torch.autograd.grad(loss(leaf, wl), (leaf, wl))
    (ref, err), (sums, es) = _gradient(gq, q, w, pos, inv, **how)
    assert (ref - want[0]).abs().max() <= 1e-12 and (sums - want[1]).abs().max() <= 1e-10
    h = 1e-3  # truncation h^2 / 6 times a third derivative (of a norm of values of size 3: below 10)
    for i in ((0, 0, 0), (3, 1, 5), (5, 0, 11), (4, 2, 17)):
        d = torch.zeros_like(leaf)
        d[i] = h
        diff = (loss(q.double() + d, w.double()) - loss(q.double() - d, w.double())) / (2 * h)
        assert abs(diff - dq[i].double()) <= err[i] + 1e-5
    for c in (0, 7, 19):  # linear in the weights: no truncation
        d = torch.zeros_like(wl)
        d[c] = 1.0
        diff = (loss(q, w.double() + d) - loss(q, w.double() - d)) / 2
        assert abs(diff - dw[c].double()) <= es[c] + 1e-10


def test_rows_of_zeros_and_large_values():
    """A head of zeros stays zero (eps keeps r finite) and its gradient is r u gz; bf16 values up to 1e18 are squared in
    fp32 without overflow."""
    from ltx_amd.kernels import rope_ops

    q, _, gq, _, w, _, pos, inv = _inputs(8, 2, 1, 64, 64, torch.bfloat16)
    q[3, 1] = 0
    q[5, 0] *= 1e17
    oq, _ = rope_ops.headnorm_rotary(q, None, w, None, pos, inv, eps=EPS)
    dq, _, _, _ = rope_ops.headnorm_rotary_grad(gq, None, q, None, w, None, pos, inv, eps=EPS)
    assert (oq[3, 1] == 0).all() and oq.isfinite().all()
    _within(oq, _forward(q, w, pos, inv))
    _within(dq, _gradient(gq, q, w, pos, inv)[0])
    q[2, 0, 5], q[4, 1, 9] = float("nan"), float("inf")
    oq, _ = rope_ops.headnorm_rotary(q, None, w, None, pos, inv, eps=EPS)
    assert oq[2, 0].isnan().all() and not oq[4, 1].isfinite().all()  # of the head they are in only
    ok = torch.ones(8, 2, dtype=torch.bool, device=DEV)
    ok[2, 0] = ok[4, 1] = False
    assert oq[ok].isfinite().all()


def test_far_heads():
    """Offsets past 2^31 elements."""
    from ltx_amd.kernels import rope_ops

    q, k, gq, gk, wq, wk, pos, inv = _inputs(5, 3, 2, 64, 64, torch.bfloat16)
    far = torch.empty(5 * (1 << 30), dtype=torch.bfloat16, device=DEV).as_strided((5, 3, 64), (1 << 30, 1 << 20, 1))
    far.copy_(q)
    a = rope_ops.headnorm_rotary(far, k, wq, wk, pos, inv, eps=EPS)
    b = rope_ops.headnorm_rotary(q, k, wq, wk, pos, inv, eps=EPS)
    c = rope_ops.headnorm_rotary_grad(gq, gk, far, k, wq, wk, pos, inv, eps=EPS, out=(far, None))
    d = rope_ops.headnorm_rotary_grad(gq, gk, q, k, wq, wk, pos, inv, eps=EPS)
    assert all(torch.equal(x, y) for x, y in zip(a + c, b + d))


def test_streams_graphs_and_empty():
    from ltx_amd.kernels import rope_ops

    q, k, gq, gk, wq, wk, pos, inv = _inputs(700, 8, 2, 128, 128, torch.bfloat16)

    def both():
        return (*rope_ops.headnorm_rotary(q, k, wq, wk, pos, inv),
                *rope_ops.headnorm_rotary_grad(gq, gk, q, k, wq, wk, pos, inv))

    want = both()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got += [both() for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for r in got for x, y in zip(r, want))
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for gr in graphs:
        with torch.cuda.graph(gr):
            outs.append(both())
    for _ in range(3):
        pos.add_(1000)
        q.copy_(torch.randn(q.shape, device=DEV))
        want = both()
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for r in outs for x, y in zip(r, want))
    none = rope_ops.headnorm_rotary(q[:0], k[:0], wq, wk, pos[:0], inv)
    assert none[0].shape == (0, 8, 128) and none[1].shape == (0, 2, 128)
    dq, dk, dwq, dwk = rope_ops.headnorm_rotary_grad(gq[:0], gk[:0], q[:0], k[:0], wq, wk, pos[:0], inv)
    assert dq.shape == (0, 8, 128) and (dwq == 0).all() and (dwk == 0).all()
    _, _, _, dwk = rope_ops.headnorm_rotary_grad(gq, gk[:, :0], q, k[:, :0], wq, wk, pos, inv)
    assert (dwk == 0).all()


def test_int8_attention_layer():
    """A run as an attention layer makes it: rows to int8, the fused query, key and value product, the per-head norm
    and rotation of the first two in place, attention, int8 again and the output projection added to the residual --
    against float64 with the roundings between the operators applied to the reference as well."""
    from ltx_amd.kernels import attention, gemm, rope_ops

    t, heads, dh = 200, 8, 64
    inner = heads * dh
    g = torch.Generator(device=DEV).manual_seed(9)
    wqkv = gemm.make_weight((torch.randn(3 * inner, 1024, generator=g, device=DEV) / 32).bfloat16(),
                            torch.randn(3 * inner, generator=g, device=DEV) * 0.1, kind="int8")
    wo = gemm.make_weight((torch.randn(1024, inner, generator=g, device=DEV) / 23).bfloat16(), kind="int8")
    nq, nk = (torch.randn(dh, generator=g, device=DEV) * 0.2 + 1 for _ in range(2))
    x = torch.randn(t, 1024, generator=g, device=DEV).bfloat16()
    gate = torch.randn(1024, generator=g, device=DEV)
    inv, _ = rope_ops.rotary_frequencies(dh)
    pos = torch.arange(t, device=DEV)
    buf = gemm.linear(gemm.quantize_rows_int8(x), wqkv)
    q, k, v = buf.split(inner, 1)
    qh, kh = q.unflatten(1, (heads, dh)), k.unflatten(1, (heads, dh))
    rope_ops.headnorm_rotary(qh, kh, nq, nk, pos, inv, eps=EPS, out=(qh, kh))
    o = attention.flash_attention(q, k, v, heads)
    y = gemm.linear(gemm.quantize_rows_int8(o), wo, epilogue=gemm.EPI_RESIDUAL, residual=x, gate=gate)
    torch.cuda.synchronize()

    def codes(a):
        s = (a.double().abs().amax(1, keepdim=True) / 127).float().double()
        return torch.round((a.double() / s).float()).double() * s

    def values(w):
        return w.w.double() * w.scale.double()[:, None]

    ref = (codes(x) @ values(wqkv).T + wqkv.bias.double()).bfloat16()
    rq, rk, rv = (a.unflatten(1, (heads, dh)) for a in ref.split(inner, 1))
    rq = _forward(rq, nq, pos, inv)[0].bfloat16().double()
    rk = _forward(rk, nk, pos, inv)[0].bfloat16().double()
    p = torch.softmax(torch.matmul(rq.transpose(0, 1), rk.permute(1, 2, 0).contiguous()) * dh ** -0.5, -1)
    ro = torch.matmul(p, rv.double().transpose(0, 1).contiguous()).transpose(0, 1).reshape(t, inner).bfloat16()
    branch = codes(ro) @ values(wo).T
    want = x.double() + gate.double() * branch
    # every operator is held to its own bound in its own test; here a rounding step of an intermediate may fall the
    # other way: 2^-8 relative for each of three bf16 stages, which moves a code of the second quantisation by at most
    # one (127 * 2^-8 < 1), and with it a value by its row's scale; the projection stretches that by its largest
    # singular value
    moved = ro.double().abs().amax(1, keepdim=True) / 127 + 3 * 2.0 ** -8 * ro.double().abs()
    stretch = torch.linalg.matrix_norm(gate.double()[:, None] * values(wo), 2)
    assert stretch * moved.norm() <= 0.5 * (gate.double() * branch).norm()  # (what a wrong operator would exceed)
    assert (y.double() - want).norm() <= stretch * moved.norm() + 2.0 ** -8 * want.norm()


@pytest.mark.parametrize("tokens", [1, 3, 30])
def test_gradient_of_few_tokens_without_a_side_or_weights(tokens):
    """Sizes around those that one workgroup per side takes: no key heads (their weights' gradient is zero, whatever the
    memory held), weights on one side only, and graphs replayed."""
    from ltx_amd.kernels import rope_ops

    q, k, gq, gk, wq, wk, pos, inv = _inputs(tokens, 8, 4, 128, 64, torch.bfloat16)
    want, sums = _gradient(gq, q, wq, pos, inv)
    for _ in range(3):
        junk = [torch.full((128,), float("nan"), device=DEV) for _ in range(8)]
        del junk
        dq, dk, dwq, dwk = rope_ops.headnorm_rotary_grad(gq, gk[:, :0], q, k[:, :0], wq, wk, pos, inv, eps=EPS)
        _within(dq, want)
        _within(dwq, sums)
        assert dk.shape == (tokens, 0, 128) and (dwk == 0).all()
    dq, dk, none, dwk = rope_ops.headnorm_rotary_grad(gq, gk, q, k, None, wk, pos, inv, eps=EPS)
    assert none is None
    _within(dq, _gradient(gq, q, None, pos, inv)[0])
    _within(dk, _gradient(gk, k, wk, pos, inv)[0])
    _within(dwk, _gradient(gk, k, wk, pos, inv)[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rope_ops.headnorm_rotary_grad(gq, gk, q, k, wq, wk, pos, inv, eps=EPS)
    for _ in range(3):
        gq.copy_(torch.randn(gq.shape, device=DEV))
        fresh = rope_ops.headnorm_rotary_grad(gq, gk, q, k, wq, wk, pos, inv, eps=EPS)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, fresh))
