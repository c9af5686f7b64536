"""Norm weights' gradients of many tokens and heads: sums of many terms a lane.

A lane adds at most 256 terms one after another in fp32, six lane exchanges and the four waves' sum follow, all else
is fp64: for terms of one sign each of the additions is off by 2^-24 of the sum so far, which grows evenly, so by
256 * 2^-25 + 8 * 2^-24 < 2^-16.9 of the result together; a term r x g by 2^-21 of itself (2^-19 where a head has many
channels, as in test_gpu_headnorm.py).  Inputs are one token's, repeated, so that a float64 result takes no memory.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("tokens,heads", [(1 << 23, 64), (1, 1 << 20), (3, 1 << 19)])
def test_equal_terms(tokens, heads):
    """4096 equal terms a lane and more, whose running fp32 sum is off to the same side at most of its steps (2^-14.1 after
    4096 of them): over many tiles, and within one."""
    from ltx_amd.kernels import rope_ops

    print(f"equal terms T={tokens} H={heads}", flush=True)
    x = torch.full((1, 1, 1), 1.6796875, dtype=torch.bfloat16, device=DEV).expand(tokens, heads, 1)
    g = torch.ones(1, 1, 1, dtype=torch.bfloat16, device=DEV).expand(tokens, heads, 1)
    w = torch.ones(1, device=DEV)
    _, _, dw, _ = rope_ops.headnorm_rotary_grad(g, None, x, None, w, None, None, None, eps=1.0)
    want = tokens * heads * 1.6796875 / (1.6796875 ** 2 + 1) ** 0.5
    assert abs(dw.double().item() / want - 1) <= 2.0 ** -16.9 + 2.0 ** -21


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,dh,rot,dtype", [
    (700000, 16, 128, 128, torch.bfloat16), (360000, 4, 510, 120, torch.float32), (180000, 16, 512, 256, torch.float16),
    (500000, 24, 80, 40, torch.bfloat16), (900000, 8, 65, 64, torch.float16), (360000, 8, 256, 64, torch.float32),
    (40000, 40, 511, 510, torch.bfloat16)])
def test_repeated_tokens(tokens, heads, dh, rot, dtype, layout):
    """Some hundred terms a lane and more in the kernel's forms: what the tokens' repetition gives is that many times one token's."""
    from ltx_amd.kernels import rope_ops

    print(f"repeated tokens T={tokens} H={heads} dh={dh} rot={rot} {dtype} {layout}", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(tokens + dh)
    q, gq = (torch.randn(1, heads, dh, generator=gen, device=DEV).to(dtype) for _ in range(2))
    k, gk = (torch.randn(1, 1, dh, generator=gen, device=DEV).to(dtype) for _ in range(2))
    w = torch.randn(dh, generator=gen, device=DEV)
    inv, _ = rope_ops.rotary_frequencies(rot)
    pos = torch.full((tokens,), 1234, device=DEV)
    one = rope_ops.headnorm_rotary_grad(gq, gk, q, k, w, w, pos[:1], inv, layout=layout)
    got = rope_ops.headnorm_rotary_grad(*(t.expand(tokens, -1, -1) for t in (gq, gk, q, k)), w, w, pos, inv, layout=layout)
    for i, (x, g) in enumerate(((q, gq), (k, gk))):
        d = got[i]
        assert torch.equal(d[0], one[i][0]) and torch.equal(d[-1], one[i][0]) and torch.equal(d[tokens // 2], one[i][0])
        v, up = x.double()[0], g.double()[0]
        n = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6)
        turn = torch.polar(torch.ones(rot // 2, dtype=torch.float64, device=DEV), -1234.0 * inv)
        z, size = up.clone(), up.abs()
        a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
        p = torch.complex(up[:, a], up[:, b]) * turn
        z[:, a], z[:, b] = p.real, p.imag
        size[:, a] = size[:, b] = up[:, a].abs() + up[:, b].abs()
        err = 2.0 ** -21 * (size * n.abs()).sum(0) + (2.0 ** -16.9 + 2.0 ** -18) * (z * n).abs().sum(0)
        over = ((got[2 + i].double() / tokens - (z * n).sum(0)).abs() - err).max().item()
        assert over <= 0, (i, over)
