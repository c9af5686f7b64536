"""MXFP4 scale words that are a column range of wider words (one projection of
several that were quantised together), up to the last word of their memory."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


# ragged against every tile height and width of the kernels
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("m,k,n", [(1, 256, 8), (5, 128, 72), (70, 1024, 264), (257, 640, 1000), (1301, 512, 4104),
                                   (2310, 384, 4360)])
def test_column_ranges_of_wider_words(m, k, n, quantised):
    from ltx_amd.kernels import gemm

    print(f"mxfp4 words M={m} K={k} N={n} quantised={quantised}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(n)
    both = gemm.quantize_rows_mxfp4(torch.randn(264 + n, k, generator=g, device=DEV))
    alone = gemm.LinearWeight("mxfp4", both.codes[264:].clone(), both.scales[:, 264:].clone())
    part = gemm.LinearWeight("mxfp4", both.codes[264:], both.scales[:, 264:])
    x = torch.randn(12 + m, k, generator=g, device=DEV).bfloat16()
    rows, own = x[12:], x[12:]
    if quantised:
        q = gemm.quantize_rows_mxfp4(x)
        rows = gemm.Mx4Rows(q.codes[12:], q.scales[:, 12:12 + m])
        own = gemm.quantize_rows_mxfp4(x[12:])
    assert torch.equal(gemm.linear(rows, part), gemm.linear(own, alone))
    if quantised:  # words whose memory ends with the rows
        words, ld = q.scales.shape
        tight = torch.empty((words - 1) * ld + m, dtype=torch.int32, device=DEV).as_strided((words, m), (ld, 1))
        tight.copy_(q.scales[:, 12:12 + m])
        assert torch.equal(gemm.linear(gemm.Mx4Rows(rows.codes, tight), part), gemm.linear(own, alone))
