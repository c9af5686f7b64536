"""The opt-in int8-activation path (``gemm.INT8_ACTIVATIONS``): which products it takes, that they are the int8
product of the quantised rows bit for bit, and a whole denoise on it.

A row's rounding: codes are off by at most half a step of max / 127, so by step / sqrt(12) in the mean square.  A row whose
largest value is at most 8 times its root mean square is then off by at most 8 / 127 / sqrt(12) = 1.8 % of it, which
moves a product's outputs by as much and costs 1.7e-4 of their cosine; the denoise is gated at 0.999 as the MXFP8
activations' (whose rounding is 2^-4 / sqrt(12) = 1.8 % of each value, at most)."""

from __future__ import annotations

import pytest
import torch

from _util import cos_sim

DEV = "cuda"


def _weight(gemm, n, k, kind="int8", seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = (torch.randn(n, k, device=DEV, generator=g) * 0.02).to(torch.bfloat16)
    return gemm.make_weight(w, torch.randn(n, device=DEV, generator=g) * 0.1, kind=kind)


def _rows(*shape, seed=2):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=g).to(torch.bfloat16)


def _same(a, b):
    return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n,epi", [(1, 2048, 2048, 0), (68, 2048, 4128, 0), (68, 8192, 2048, 2), (700, 1024, 520, 1),
                                       (1296, 4096, 4096, 3), (3456, 4096, 12320, 0)])
def test_the_switch_takes_int8_weights_only(monkeypatch, m, k, n, epi):
    from ltx_amd.kernels import gemm

    print(f"int8 activations M={m} K={k} N={n} epi={epi}", flush=True)
    weight, x = _weight(gemm, n, k), _rows(m, k)
    how = dict(epilogue=epi)
    if epi in (gemm.EPI_RESIDUAL, gemm.EPI_RESIDUAL_ROUND):
        how.update(residual=_rows(m, n, seed=3), gate=torch.rand(n, device=DEV))
    elif epi == gemm.EPI_BIAS and n % 64 == 32:
        how.update(sigmoid_from=n - 32)
    plain = gemm.linear(x, weight, **how)
    want = gemm.linear(gemm.quantize_rows_int8(x), weight, **how)
    eligible = gemm.rowss_eligible(x, weight)
    monkeypatch.setattr(gemm, "INT8_ACTIVATIONS", True)
    got = gemm.linear(x, weight, **how)
    explicit = gemm.linear(x, weight, splits=1, **how)  # a call that asks for the other kernels' way gets it
    assert eligible == (m == 3456) and not gemm.rowss_eligible(x, weight)
    mx = _weight(gemm, n, k, "mxfp8") if k % 512 == 0 else None
    on = None if mx is None else gemm.linear(x, mx, **how)
    monkeypatch.setattr(gemm, "INT8_ACTIVATIONS", False)
    off = None if mx is None else gemm.linear(x, mx, **how)
    again = gemm.linear(x, weight, **how)
    torch.cuda.synchronize()
    assert _same(got, want) and not _same(got, plain) and _same(again, plain)
    assert mx is None or _same(on, off)
    assert explicit.shape == plain.shape and not _same(explicit, got)


@pytest.mark.gpu
def test_leading_axes_outputs_and_no_rows(monkeypatch):
    from ltx_amd.kernels import gemm

    weight = _weight(gemm, 520, 1024)
    x, res, gate = _rows(3, 37, 1024), _rows(3, 37, 520, seed=3), torch.rand(520, device=DEV)
    monkeypatch.setattr(gemm, "INT8_ACTIVATIONS", True)
    flat = gemm.linear(x.view(111, 1024), weight, epilogue=gemm.EPI_RESIDUAL, residual=res.view(111, 520), gate=gate)
    y = gemm.linear(x, weight, epilogue=gemm.EPI_RESIDUAL, residual=res, gate=gate)
    assert y.shape == (3, 37, 520) and _same(y.view(111, 520), flat)
    wide = torch.full((111, 640), 7.0, device=DEV, dtype=torch.bfloat16)
    out = wide.view(3, 37, 640)[:, :, 64:584]
    gemm.linear(x, weight, epilogue=gemm.EPI_RESIDUAL, residual=res, gate=gate, out=out)
    gemm.linear(x, weight, epilogue=gemm.EPI_RESIDUAL, residual=res, gate=gate, out=res)  # in place
    torch.cuda.synchronize()
    assert _same(out, y) and _same(res, y) and bool((wide[:, :64] == 7).all()) and bool((wide[:, 584:] == 7).all())
    one = gemm.linear(x[0, 0], weight)
    assert one.shape == (520,) and _same(one, gemm.linear(x[0, :1], weight)[0])
    assert gemm.linear(x[:, :0], weight).shape == (3, 0, 520)
    with pytest.raises(ValueError):
        gemm.linear(x, weight, out=torch.empty(111, 520, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(ValueError):  # rows that no stride gives
        gemm.linear(x, weight, out=torch.empty(37, 3, 520, device=DEV, dtype=torch.bfloat16).transpose(0, 1))


@pytest.mark.gpu
def test_eight_steps_four_blocks_vs_oracle(monkeypatch):
    """A 4-block full-width int8 model on 384 video tokens, every projection on int8 rows, against the oracle's
    bf16-activation arithmetic, per step; and the first step captured and replayed against the eager one."""
    from test_gpu_model import _model_weights

    from ltx_amd.kernels import gemm
    from ltx_amd.model.transformer.model import LTXModel
    from ltx_amd.pipeline import DenoiseState, denoise
    from oracle import block as ob
    from oracle import rope as orope

    print("int8 activations: 4-block int8 model, 384 video tokens, 8 steps vs oracle", flush=True)
    monkeypatch.setattr(gemm, "INT8_ACTIVATIONS", True)
    taken, fn = [], gemm._linear_int8
    monkeypatch.setattr(gemm, "_linear_int8", lambda x, *a: (taken.append(x.shape[0]), fn(x, *a))[1])
    model = LTXModel(num_layers=4, weight_format="int8", seed=21)
    st = DenoiseState(model, height=256, width=384, frames=25, text_tokens=256, audio_frames=26, seed=7)
    weights = _model_weights(model)
    vlat, alat = st.video_latent.float().cpu(), st.audio_latent.float().cpu()
    vctx, actx = st.video_context.float().cpu(), st.audio_context.float().cpu()
    vpos, apos = st.video_positions, st.audio_positions
    pes = tuple(tuple(torch.from_numpy(a) for a in p) for p in (
        orope.rope_tables(vpos, 4096, 32, orope.VIDEO_MAX_POS),
        orope.rope_tables(vpos[:, 0:1], 2048, 32, orope.AUDIO_MAX_POS),
        orope.rope_tables(apos, 2048, 32, orope.AUDIO_MAX_POS),
        orope.rope_tables(apos[:, 0:1], 2048, 32, orope.AUDIO_MAX_POS)))
    got = []
    denoise(model, st, callback=lambda step, s: got.append(
        (s.video_latent.float().cpu().clone(), s.audio_latent.float().cpu().clone())))
    # per block and step of the video rows: QKV, out, text query and out, the cross-attentions', feed-forward up and down
    assert taken.count(384) >= 8 * 4 * 8 and taken.count(26) >= 8 * 4 * 8
    for step in range(8):
        vlat, alat = ob.model_step(weights, vlat, alat, vctx, actx, st.sigmas[step], st.sigmas[step + 1], pes)
        cv, ca = cos_sim(got[step][0].numpy(), vlat.numpy()), cos_sim(got[step][1].numpy(), alat.numpy())
        print(f"int8 step {step}: video cos {cv:.6f} audio cos {ca:.6f}", flush=True)
        assert cv >= 0.999 and ca >= 0.999


@pytest.mark.gpu
def test_a_step_captured_and_replayed(monkeypatch):
    """A step with its audio stream beside the video's, in one graph, equals the eager one at every replay."""
    from ltx_amd.kernels import gemm
    from ltx_amd.model.transformer.model import LTXModel
    from ltx_amd.pipeline import DenoiseState, denoise_step

    print("int8 activations: a captured step", flush=True)
    monkeypatch.setattr(gemm, "INT8_ACTIVATIONS", True)
    model = LTXModel(num_layers=2, weight_format="int8", seed=5)
    st = DenoiseState(model, height=256, width=384, frames=25, text_tokens=256, audio_frames=26, seed=7)
    pes = model.rope(st.video_positions, st.audio_positions)
    start = st.video_latent.clone(), st.audio_latent.clone()

    def reset():
        st.video_latent.copy_(start[0])
        st.audio_latent.copy_(start[1])

    denoise_step(model, st, 0, pes)
    torch.cuda.synchronize()
    want = st.video_latent.clone(), st.audio_latent.clone()
    reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        denoise_step(model, st, 0, pes)
    for _ in range(3):
        reset()
        graph.replay()
        torch.cuda.synchronize()
        assert _same(st.video_latent, want[0]) and _same(st.audio_latent, want[1])


def test_which_products_the_switch_takes(monkeypatch):
    from ltx_amd.kernels import gemm

    def weight(kind, k=128):
        return gemm.LinearWeight(kind=kind, w=torch.empty((64, k), dtype=torch.int8))

    x = torch.empty((4, 128), dtype=torch.bfloat16)
    assert not gemm._int8_eligible(x, weight("int8"), gemm.TILE_AUTO, None)  # off by default
    monkeypatch.setattr(gemm, "INT8_ACTIVATIONS", True)
    assert gemm._int8_eligible(x, weight("int8"), gemm.TILE_AUTO, None)
    assert gemm._int8_eligible(x, weight("int8"), gemm.TILE_G8, None)
    assert not gemm._int8_eligible(x, weight("int8"), gemm.TILE_128, None)
    assert not gemm._int8_eligible(x, weight("int8"), gemm.TILE_AUTO, 2)
    assert not gemm._int8_eligible(x.float(), weight("int8"), gemm.TILE_AUTO, None)
    assert not gemm._int8_eligible(x, weight("mxfp8"), gemm.TILE_AUTO, None)
    assert not gemm._int8_eligible(x, weight("int8", 96), gemm.TILE_AUTO, None)
    assert not gemm._int8_eligible(x, weight("int8", 1 << 17), gemm.TILE_AUTO, None)
