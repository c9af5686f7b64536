"""MXFP4 weights and scale words whose rows lie so far apart that byte offsets pass
31 bits: what the tile kernels take goes to the kernel with 64-bit addresses, with
and without K ranges, and quantised rows are refused; the results are those of the
same weights close together."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("what", ["codes", "words"])
# one row; K ranges of the mid-size kernel; one pass of it; 128-row tiles and whole rounds of the 8-wave kernel
@pytest.mark.parametrize("m,k,n", [(1, 4096, 2048), (68, 8192, 2048), (300, 1024, 2056), (1296, 704, 4096),
                                   (3456, 640, 4096)])
def test_weights_past_two_gib(m, k, n, what):
    from ltx_amd import _lib
    from ltx_amd.kernels import gemm

    print(f"mxfp4 far {what} M={m} K={k} N={n}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(m + n)
    near = gemm.quantize_rows_mxfp4(torch.randint(-8, 9, (n, k), generator=g, device=DEV).float())
    codes, words = near.codes, near.scales
    if what == "codes":
        stride = ((1 << 31) // n + 16) // 16 * 16
        codes = torch.zeros(n, stride, dtype=torch.uint8, device=DEV)[:, :k // 2]
        codes.copy_(near.codes)
        assert (n - 1) * codes.stride(0) + k // 2 > (1 << 31) - stride and n * codes.stride(0) >= 1 << 31
    else:
        rows = words.shape[0]
        stride = ((1 << 29) // rows + 4) // 4 * 4
        words = torch.zeros(rows, stride, dtype=torch.int32, device=DEV)[:, :n]
        words.copy_(near.scales[:, :n])
        assert rows * words.stride(0) >= 1 << 29
    # small whole numbers: every sum is exact, whichever kernel and K ranges make it
    x = torch.randint(-8, 9, (m, k), generator=g, device=DEV).bfloat16()
    bias = torch.randint(-8, 9, (n,), generator=g, device=DEV).float()
    res, gate = torch.randn(m, n, generator=g, device=DEV).bfloat16(), torch.randn(n, generator=g, device=DEV)
    here, there = (gemm.LinearWeight("mxfp4", c, s, bias) for c, s in ((near.codes, near.scales), (codes, words)))
    for kw in (dict(), dict(epilogue=gemm.EPI_GELU), dict(epilogue=gemm.EPI_RESIDUAL, residual=res, gate=gate)):
        assert torch.equal(gemm.linear(x, there, **kw), gemm.linear(x, here, **kw)), kw
    if k % 128 == 0:
        with pytest.raises(_lib.LtxKernelError):
            gemm.linear(gemm.quantize_rows_mxfp4(x), there)
