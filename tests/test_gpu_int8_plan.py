"""int8 products of sizes that the plan splits: rows of whole rounds in one launch and the rest in another, and K
ranges; every kernel that such a launch can be.  test_int8_plan_host.py checks that these sizes (with those of
test_gpu_int8.py) reach them all.  Bounds: test_gpu_int8.py."""

from __future__ import annotations

import pytest
import torch

import test_gpu_int8 as base

pytestmark = pytest.mark.gpu
DEV = "cuda"

# the rest on tiles; on the few-row kernel; heads of 128 columns
TWO_LAUNCHES = [(590, 26576, 320), (1477, 12744, 512), (1172, 16384, 512), (652, 22312, 2304), (4899, 30104, 960),
                (12155, 1304, 192), (5120, 4096, 4096), (1497, 12744, 4032),
                (2331, 8192, 256), (14969, 1032, 128), (913, 16752, 192),
                (1870, 10760, 2752), (801, 27208, 1856), (15631, 1048, 1216), (18697, 776, 384), (1552, 10832, 512),
                (2073, 3864, 1984), (1556, 10824, 448), (18879, 808, 320), (594, 16256, 16256)]
RANGES = [(33, 8, 2752), (133, 3424, 24576), (1392, 8, 3520), (351, 3840, 16000), (4624, 8, 6592), (485, 9720, 16000),
          (8540, 136, 13632), (1025, 4096, 16384), (8423, 144, 17408)]
ONE_LAUNCH = [(1, 8192, 256), (9, 12888, 320), (25, 8200, 192), (40, 8256, 128), (386, 7112, 128), (579, 8152, 128),
              (16969, 392, 128), (10896, 1368, 64), (65, 7624, 384)]


@pytest.mark.parametrize("m,n,k", TWO_LAUNCHES + RANGES + ONE_LAUNCH)
def test_products(m, n, k):
    """Every epilogue against float64, and the residual in place."""
    from ltx_amd.kernels import gemm

    base.test_products(m, n, k)
    rows, weight = base._case(m, n, k)
    g = torch.Generator(device=DEV).manual_seed(4)
    residual = torch.randn(m, n, generator=g, device=DEV).bfloat16()
    gate = torch.randn(n, generator=g, device=DEV)
    for epilogue in (gemm.EPI_RESIDUAL, gemm.EPI_RESIDUAL_ROUND):
        want = gemm.linear(rows, weight, epilogue=epilogue, residual=residual, gate=gate)
        into = residual.clone()
        assert gemm.linear(rows, weight, epilogue=epilogue, residual=into, gate=gate, out=into) is into
        assert torch.equal(into, want)


@pytest.mark.parametrize("m,n,k", [(1172, 16384, 512), (2331, 8192, 256), (1552, 10832, 512), (351, 3840, 16000)])
def test_strided_rows(m, n, k):
    """Activations, outputs and residual as columns of wider buffers: the second launch starts at their strides."""
    from ltx_amd.kernels import gemm

    rows, weight = base._case(m, n, k)
    wide = torch.zeros(m, k + 32, dtype=torch.int8, device=DEV)
    wide[:, 16:k + 16] = rows.codes
    buf = torch.full((m, n + 24), 7.0, device=DEV).bfloat16()
    residual = torch.randn(m, n + 16, device=DEV).bfloat16()[:, 8:n + 8]
    gate = torch.randn(n, device=DEV)
    kw = dict(epilogue=gemm.EPI_RESIDUAL, residual=residual, gate=gate)
    got = gemm.linear(gemm.Int8Rows(wide[:, 16:k + 16], rows.scales), weight, out=buf[:, 8:n + 8], **kw)
    assert torch.equal(got, gemm.linear(rows, weight, **kw))
    assert (buf[:, :8] == 7.0).all() and (buf[:, n + 8:] == 7.0).all()


# one launch of tiles, K ranges and two launches by size; weights, or a tile's rows, past 31 bits of byte offsets
@pytest.mark.parametrize("m,n,k,ldw", [(200, 72, 320, (1 << 25) + 16), (130, 264, 8192, 1 << 23), (913, 16752, 192, 1 << 18)])
def test_far_weights(m, n, k, ldw):
    """Tiles address weights with 31 bits: larger ones go to the few-row kernel."""
    from ltx_amd.kernels import gemm

    print(f"far weights {m} x {k} -> {n}, stride {ldw}", flush=True)
    rows, weight = base._case(m, n, k)
    assert n * ldw > 1 << 31
    far = torch.empty(n * ldw, dtype=torch.int8, device=DEV).as_strided((n, k), (ldw, 1))
    far.copy_(weight.w)
    got = gemm.LinearWeight("int8", far, weight.scale, weight.bias)
    res, gate = torch.randn(m, n, device=DEV).bfloat16(), torch.randn(n, device=DEV)
    for kw in (dict(), dict(epilogue=gemm.EPI_GELU), dict(epilogue=gemm.EPI_RESIDUAL, residual=res, gate=gate)):
        assert torch.equal(gemm.linear(rows, got, **kw), gemm.linear(rows, weight, **kw))


@pytest.mark.parametrize("m,n,k", [(300, 264, 320), (300, 264, 8192)])
def test_rows_too_far_apart_for_a_tile(m, n, k):
    from ltx_amd.kernels import gemm

    lda = (1 << 23) + 16
    print(f"far rows {m} x {k} -> {n}, stride {lda}", flush=True)
    rows, weight = base._case(m, n, k)
    far = torch.empty(m * lda, dtype=torch.int8, device=DEV).as_strided((m, k), (lda, 1))
    far.copy_(rows.codes)
    assert torch.equal(gemm.linear(gemm.Int8Rows(far, rows.scales), weight), gemm.linear(rows, weight))
