"""The gated residual of MXFP4 products: fp32 from the sum to the output.

Operands are small multiples of 1/2, so every partial sum is a multiple of 1/4
below 2^22 and exact in fp32 in any order: what remains are the roundings of
the epilogue.  The residual is about minus the branch, so that a rounding of
the branch (2^-8 of it) is as large as the result itself.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = 2.0 ** -8
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)

# (M, K, N) for every kernel: one to 16 rows; K ranges and the joining launch; depths that end inside a scale
# word; 64, 128, 192 rows of the mid-size tiles; 128- and 256-row tiles of the 8-wave kernel; whole rounds and
# the rows left over; the four tile shapes of quantised rows
SHAPES = [(1, 4096, 4096), (16, 2048, 264), (3, 192, 72), (68, 8192, 2048), (68, 8128, 520), (50, 320, 136),
          (256, 4096, 1024), (300, 1024, 712), (1296, 4096, 4096), (1296, 704, 4096), (1300, 512, 12320),
          (3456, 1024, 4104)]


def _rows(rows, k, g):
    nib = torch.randint(0, 16, (rows, k), generator=g, device=DEV, dtype=torch.uint8)
    words = torch.full(((k + 127) // 128, (rows + 3) // 4 * 4), 0x7f7f7f7f, dtype=torch.int32, device=DEV)
    return nib[:, ::2] | nib[:, 1::2] << 4, words, torch.tensor(E2M1, device=DEV)[nib.int()].double()


@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_branch_is_not_rounded(m, k, n, quantised):
    from ltx_amd.kernels import gemm

    if quantised and k % 128:
        pytest.skip("K is no multiple of 128")
    print(f"mxfp4 residual M={m} K={k} N={n} quantised={quantised}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(m + n)
    wc, ws, w = _rows(n, k, g)
    if quantised:
        xc, xs, xv = _rows(m, k, g)
        x = gemm.Mx4Rows(xc, xs)
    else:
        xv = torch.randint(-8, 9, (m, k), generator=g, device=DEV).double()
        x = xv.bfloat16()
    bias = torch.randint(-64, 65, (n,), generator=g, device=DEV) / 2
    gate = torch.randn(n, generator=g, device=DEV)
    acc = xv @ w.T
    assert acc.abs().max() < 2 ** 22
    for qlinear in (False, True):
        y = (acc.bfloat16().double() if qlinear else acc) + bias.double()
        res = (-gate.double() * y).bfloat16()
        wt = gemm.LinearWeight("mxfp4", wc, ws, bias, qlinear=qlinear)
        got = gemm.linear(x, wt, epilogue=gemm.EPI_RESIDUAL, residual=res, gate=gate)
        want = res.double() + gate.double() * y
        # one fp32 rounding (the fused product and sum), one to bf16
        over = (got.double() - want).abs() - (HALF * (1 + 2.0 ** -20) + 2.0 ** -23) * want.abs()
        assert over.max().item() <= 0, ((over > 0).float().mean().item(), over.max().item())
        # the form that rounds: each step of it as torch does it
        got = gemm.linear(x, wt, epilogue=gemm.EPI_RESIDUAL_ROUND, residual=res, gate=gate)
        branch = (gate * y.float().bfloat16().float()).bfloat16()
        assert torch.equal(got, (res.float() + branch.float()).bfloat16())
