"""MXFP4 as a resident weight format: a block's forward against the oracle on
the decoded weights, the FP8 checkpoint loader's fused rows, a captured step."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import _cache_fixture as fx
from oracle import quant as oq
from test_gpu_block import _gate, _run
from test_gpu_transformer_cache import _fused_parts, _small_model, _small_W

pytestmark = pytest.mark.gpu


def test_av_block_on_mxfp4_weights():
    gv, rv, ga, ra = _run("mxfp4", (3, 8, 12), 20, seed=3)
    _gate(gv, rv, "mxfp4 video")
    _gate(ga, ra, "mxfp4 audio")


def test_checkpoint_loads_as_mxfp4(tmp_path):
    """Each projection of a fused weight keeps its own blocks; loading again
    reuses the storage."""
    from ltx_amd.kernels import gemm
    from ltx_amd.loader import load_transformer_weights

    W = _small_W(seed=2)
    p = tmp_path / "ltx-fp8.safetensors"
    fx.write_safetensors(p, fx.checkpoint_items(W, fp8=True))
    model = _small_model(fmt="mxfp4")
    load_transformer_weights(model, p, weight_format="mxfp4")
    before = model.transformer_blocks[0].attn1.proj_q
    load_transformer_weights(model, p, weight_format="mxfp4")
    assert model.transformer_blocks[0].attn1.proj_q.w.data_ptr() == before.w.data_ptr()
    for lw, parts in _fused_parts(model.transformer_blocks[0], 0):
        assert lw.kind == "mxfp4" and not lw.qlinear
        enc = [oq.mxfp4_quantize(W["linears"][q]["w"]) for q in parts]
        codes, scales = (np.concatenate([e[i] for e in enc]) for i in (0, 1))
        b, w = oq.mxfp4_pack(codes, scales)
        n = codes.shape[0]
        np.testing.assert_array_equal(lw.w.cpu().numpy(), b, err_msg=parts[0])
        np.testing.assert_array_equal(lw.scale.cpu().numpy()[:, :n], w[:, :n], err_msg=parts[0])
        want = torch.from_numpy(oq.mxfp4_dequantize(codes, scales)).bfloat16()
        assert torch.equal(gemm.dequantize(lw).cpu(), want)


def test_projection_refuses_non_matching_rows():
    from ltx_amd.kernels import gemm

    w8 = gemm.make_weight(torch.randn(64, 128, device="cuda").bfloat16(), kind="mxfp8")
    w4 = gemm.make_weight(torch.randn(64, 128, device="cuda").bfloat16(), kind="mxfp4")
    x = torch.randn(4, 128, device="cuda").bfloat16()
    with pytest.raises(ValueError):
        gemm.linear(gemm.quantize_rows_mxfp4(x), w8)
    with pytest.raises(ValueError):
        gemm.linear(gemm.MxRows(*gemm.quantize_rows_mxfp8(x)), w4)
    with pytest.raises(ValueError):
        gemm.linear_mx(*gemm.quantize_rows_mxfp8(x), w4)
    with pytest.raises(ValueError):
        gemm.linear(x, w4, out=torch.empty(4, 64, device="cuda"))
