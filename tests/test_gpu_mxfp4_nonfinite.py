"""An infinite activation of an MXFP4 product spoils its whole row: infinity times
any E2M1 value is infinite or NaN."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "mx"])
# each kernel: one row, few rows (K ranges; a depth inside a scale word), mid-size and 8-wave tiles
@pytest.mark.parametrize("m,k,n", [(1, 768, 64), (16, 4096, 264), (68, 8192, 2048), (90, 704, 200), (300, 1024, 712),
                                   (1300, 512, 12320), (2000, 768, 4096)])
def test_rows_of_a_non_finite_activation(m, k, n, quantised, bad):
    from ltx_amd.kernels import gemm

    if quantised and k % 128:
        pytest.skip("K is no multiple of 128")
    g = torch.Generator(device=DEV).manual_seed(m)
    w = gemm.make_weight(torch.randn(n, k, generator=g, device=DEV).bfloat16(), kind="mxfp4")
    x = torch.randn(m, k, generator=g, device=DEV).bfloat16()
    rows = sorted({0, m // 2, m - 1})
    for i, r in enumerate(rows):
        x[r, (i * k // 2) % k] = bad
    got = gemm.linear(gemm.quantize_rows_mxfp4(x) if quantised else x, w)
    assert not torch.isfinite(got[rows]).any()
    keep = torch.ones(m, dtype=torch.bool, device=DEV)
    keep[rows] = False
    assert torch.isfinite(got[keep]).all()
