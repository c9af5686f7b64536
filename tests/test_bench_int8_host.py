"""bench.py and the launch observer with int8 activations: products of int8 rows are named, and measured against the
int8 MFMA's peak, with what quantises their rows inside the observed span (no GPU needed)."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import bench  # noqa: E402


def test_the_dominant_kernel_is_the_one_that_ran():
    r = bench.ff_up_roofline("w8a8", 3456, 0.200, 8, "stamps")
    assert r["peak"] == bench.PEAK_INT8_TOPS == 2 * bench.PEAK_BF16_TFLOPS and r["traffic"] is None
    assert "gemm_i8_kernel" in r["kernel"] and "int8 MFMA" in r["kernel"] and "bf16" not in r["kernel"]
    assert r["frac"] == pytest.approx(2 * 3456 * 4096 * 16384 / 0.2e-3 / 5e15, abs=1e-4)
    for kind in ("mxfp8", "int8", "bf16"):
        r = bench.ff_up_roofline(kind, 3456, 0.4, 8, "stamps")
        assert r["peak"] == bench.PEAK_BF16_TFLOPS and f"gemm8_kernel<{kind},GELU>" in r["kernel"]
        assert "bf16 MFMA" in r["kernel"] and r["unit"] == "TFLOP/s"
        assert r["traffic"] == bench.measured_traffic(f"gemm8_kernel<{kind},GELU>", kind)


def test_classes_are_measured_against_their_own_peak():
    shapes = {"ff_up": (16384, 4096), "ff_down": (4096, 16384), "qkv": (12320, 4096), "out": (4096, 4096),
              "text_q": (4128, 4096), "a2v_q": (2080, 4096), "a2v_out": (4096, 2048)}
    for kind, name, other, peak in (("w8a8", "frac_int8_peak", "frac_bf16_peak", bench.PEAK_INT8_TOPS),
                                    ("int8", "frac_bf16_peak", "frac_int8_peak", bench.PEAK_BF16_TFLOPS)):
        summary = bench.gemm_class_summary([(c, (kind, 3456, n, k, 0), 0.25) for c, (n, k) in shapes.items()])
        assert set(summary) == {*shapes, "video_stream"}
        for c in summary.values():
            assert other not in c and c[name] == pytest.approx(c["tflops"] / peak, abs=1e-3)
    # launches with different peaks have no fraction in common
    mixed = bench.gemm_class_summary([("audio", (kind, 68, 2048, 2048, 0), 0.25) for kind in ("w8a8", "bf16")])["audio"]
    assert mixed["launches"] == 2 and "frac_bf16_peak" not in mixed and "frac_int8_peak" not in mixed


def test_the_observer_spans_the_rows_quantisation(monkeypatch):
    """pre, the quantiser, the product, post; the product alone where its rows come quantised."""
    from ltx_amd import _lib
    from ltx_amd.kernels import gemm

    if not _lib.LIB_PATH.exists():
        pytest.skip("libltx_hip.so not built")
    _lib.lib()
    seen = []
    rows = gemm.Int8Rows(torch.zeros(6, 128, dtype=torch.int8), torch.zeros(6))
    weight = gemm.LinearWeight("int8", torch.zeros(64, 128, dtype=torch.int8), torch.zeros(64))
    monkeypatch.setattr(_lib, "CALLS", None)
    monkeypatch.setattr(_lib, "same_device", lambda *t: 0)
    monkeypatch.setattr(_lib, "launch", lambda device, name, *a: (seen.append(name), 0)[1])
    monkeypatch.setattr(gemm, "quantize_rows_int8", lambda x: (seen.append("rows"), rows)[1])
    monkeypatch.setattr(gemm, "LAUNCH_HOOK", lambda phase, info: seen.append((phase, info)))
    monkeypatch.setattr(gemm, "INT8_ACTIVATIONS", True)
    info = ("w8a8", 6, 64, 128, gemm.EPI_GELU)
    product = "ltx_gemm_i8_bf16"
    for x, out in ((torch.zeros(6, 128), None), (torch.zeros(2, 3, 128), None),
                   (torch.zeros(2, 3, 128), torch.empty(2, 3, 64, dtype=torch.bfloat16))):
        del seen[:]
        y = gemm.linear(x.bfloat16(), weight, epilogue=gemm.EPI_GELU, out=out)
        assert y.shape == (*x.shape[:-1], 64) and (out is None or y is out)
        assert seen == [("pre", info), "rows", product, ("post", info)]
    del seen[:]
    gemm.linear(rows, weight, epilogue=gemm.EPI_GELU)
    assert seen == [("pre", info), product, ("post", info)]
