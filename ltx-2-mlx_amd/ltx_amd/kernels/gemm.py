"""Projection GEMMs: ``y = epilogue(x @ W.T + b)`` on gfx950 matrix cores.

One entry point, :func:`linear`, for the resident weight formats of
:class:`LinearWeight` (bf16, int8 W8A16, MXFP8, MXFP4).  It replaces ``nn.Linear`` /
``mx.addmm`` (model/transformer/attention.py:425-437,
feed_forward.py:91-112) and ``mx.quantized_matmul`` for the mxfp8 cache
(loader/transformer_cache.py:177-193).  The epilogues fuse what the reference
evaluates right after the projection:

* ``EPI_BIAS``            ``bf16(x W^T + b)``
* ``EPI_GELU``            ``bf16(gelu_tanh(bf16(x W^T + b)))`` (feed_forward.py:101-102)
* ``EPI_RESIDUAL``        ``bf16(res + gate * bf16(x W^T + b))``, the gated residual add
                          of fused_ops.py:345-348 / transformer.py:598, :625
* ``EPI_RESIDUAL_ROUND``  ``bf16(res + bf16(gate * bf16(x W^T + b)))`` (transformer.py:387, :484)
* ``EPI_SIGMOID2``        ``bf16(2 * bf16(sigmoid(bf16(x W^T + b))))``, the per-head gate
                          (attention.py:563-569)

Opt-in (``MX_ACTIVATIONS``, environment ``LTX_MX_ACTIVATIONS=1``): MXFP8
weights multiply MXFP8-quantised activations on the scaled fp8 MFMA
(:func:`linear_mx`) instead of bf16 activations.  That is not the reference's
arithmetic -- its MXFP8 path keeps the activations in bf16 -- and the
activations' E4M3 rounding moves outputs by a few percent of their range.

MXFP4 (E2M1 codes, an E8M0 scale per 32 along K; the reference has it as a
quantisation mode of its feed-forward cache, which is not read): weights at
half MXFP8's bytes, times bf16 activations in :func:`linear`, or times MXFP4
activations (:class:`Mx4Rows`, from :func:`quantize_rows_mxfp4`) on the scaled
FP4 MFMA.  Its GELU, head gate and ``EPI_RESIDUAL`` act on the fp32 value,
without the bf16 rounding before them.

int8 weights take int8 activations as well (:class:`Int8Rows`, a scale per
row, from :func:`quantize_rows_int8`): the int8 MFMA at twice the bf16 rate,
exact int32 sums, epilogues on the fp32 value as MXFP4's.  Opt-in
(``INT8_ACTIVATIONS``, environment ``LTX_INT8_ACTIVATIONS=1``): :func:`linear`
quantises bf16 rows for every int8 weight, as the model's projections use it;
not the reference's arithmetic either.
"""

from __future__ import annotations

import functools
import os
from dataclasses import dataclass

import torch

from .. import _lib

EPI_BIAS = _lib.GEMM_EPI_BIAS
EPI_GELU = _lib.GEMM_EPI_GELU
EPI_RESIDUAL = _lib.GEMM_EPI_RESIDUAL
EPI_RESIDUAL_ROUND = _lib.GEMM_EPI_RESIDUAL_ROUND
EPI_SIGMOID2 = _lib.GEMM_EPI_SIGMOID2
TILE_AUTO, TILE_256, TILE_128, TILE_256_DMA, TILE_256x128, TILE_G8, TILE_G8_128 = 0, 1, 2, 3, 4, 5, 6


FORMATS = ("bf16", "int8", "mxfp8", "mxfp4")

# Opt-in quantised-activation path for MXFP8 weights (see the module text):
# products with at least this many 256x256 tiles quantise their activations
# and run ltx_gemm_mx_bf16.
MX_ACTIVATIONS = os.environ.get("LTX_MX_ACTIVATIONS", "0") == "1"
MX_MIN_TILES = 100

# The same for int8 weights, at all sizes: quantising the rows and the int8
# product take less than the bf16 rows' product at every projection of the
# model (us, weights from HBM): 16 x 2048 -> 2048 7.9 / 10.9, 68 x 8192 -> 2048
# 18.9 / 19.1, 3456 x 4096 -> 16384 217 / 391, 3456 x 16384 -> 4096 216 / 374.
INT8_ACTIVATIONS = os.environ.get("LTX_INT8_ACTIVATIONS", "0") == "1"

# Optional launch observer: called as hook(phase, info) with phase "pre" /
# "post" around every GEMM launch on the launching stream (used by bench.py
# to time chosen launches with stream events), what quantises its rows
# included.  info: (weight format, "w8a8" where int8 rows meet int8 weights;
# M, N, K, epilogue).  None in normal operation.
LAUNCH_HOOK = None


@dataclass
class LinearWeight:
    """A projection weight resident in HBM.

    ``w`` is (N, K) in nn.Linear layout: bf16, int8 codes, or E4M3 codes
    (uint8).  ``scale`` is fp32 (N) for int8 and E8M0 uint8 (N, K/32) for
    mxfp8.  ``bias`` is fp32 (N) or None.  mxfp4: ``w`` is (N, K/2) uint8, two
    E2M1 codes per byte, the even k low, and ``scale`` int32 words
    (ceil(K/128), N rounded up to 4), word [k/128, n] the E8M0 bytes of row n's
    four blocks of those 128 k (:func:`mxfp4_scale_words`).

    ``qlinear`` selects the reference module whose arithmetic the GEMM
    reproduces: False for ``nn.Linear`` (``mx.addmm``: bias added to the fp32
    accumulator, one rounding), True for ``nn.QuantizedLinear`` /
    ``_PretransposedQuantizedLinear`` (loader/transformer_cache.py:177-193:
    ``quantized_matmul(x, w) + bias``, the product rounded to bf16 before the
    bias add).  MXFP8 weights are the reference's quantised linears, so
    ``make_weight(kind="mxfp8")`` sets it; a quantised cache weight decoded
    to bf16 keeps it.
    """

    kind: str
    w: torch.Tensor
    scale: torch.Tensor | None = None
    bias: torch.Tensor | None = None
    qlinear: bool = False

    @property
    def out_features(self) -> int:
        return self.w.shape[0]

    @property
    def in_features(self) -> int:
        return self.w.shape[1] * (2 if self.kind == "mxfp4" else 1)

    def nbytes(self) -> int:
        n = self.w.numel() * self.w.element_size()
        for t in (self.scale, self.bias):
            if t is not None:
                n += t.numel() * t.element_size()
        return n


def _quantize(kind: str, w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    n, k = w.shape
    w = w.contiguous()
    stream = _lib.stream_of(w)
    if kind == "int8":
        q = torch.empty((n, k), dtype=torch.int8, device=w.device)
        s = torch.empty((n,), dtype=torch.float32, device=w.device)
        _lib.call("ltx_quantize_w8_bf16", w.data_ptr(), k, n, k, q.data_ptr(), k, s.data_ptr(), stream,
                  detail=f"N={n} K={k}")
        return q, s
    if kind == "mxfp8":
        q = torch.empty((n, k), dtype=torch.uint8, device=w.device)
        s = torch.empty((n, k // 32), dtype=torch.uint8, device=w.device)
        _lib.call("ltx_quantize_mxfp8_bf16", w.data_ptr(), k, n, k, q.data_ptr(), k, s.data_ptr(), k // 32,
                  stream, detail=f"N={n} K={k}")
        return q, s
    if kind == "mxfp4":
        rows = quantize_rows_mxfp4(w)
        return rows.codes, rows.scales
    raise ValueError(f"unknown quantised format {kind!r}")


def make_weight(w: torch.Tensor, bias: torch.Tensor | None = None, kind: str = "bf16") -> LinearWeight:
    """Build a resident weight from a bf16 (N, K) device tensor.

    ``kind="int8"`` / ``"mxfp8"`` / ``"mxfp4"`` quantise on the device with the library's
    encoders (include/ltx_hip.h "weight formats").
    """
    if w.dtype != torch.bfloat16 or w.dim() != 2 or not w.is_cuda:
        raise ValueError("make_weight expects a 2-D bf16 device tensor")
    b = None if bias is None else bias.detach().to(device=w.device, dtype=torch.float32).contiguous()
    if kind == "bf16":
        return LinearWeight("bf16", w.contiguous(), None, b)
    q, s = _quantize(kind, w)
    return LinearWeight(kind, q, s, b, qlinear=kind == "mxfp8")


def dequantize(weight: LinearWeight) -> torch.Tensor:
    """bf16 (N, K) values of a weight, decoded exactly per its format."""
    if weight.kind == "mxfp4":
        return dequantize_rows_mxfp4(Mx4Rows(weight.w, weight.scale))
    n, k = weight.w.shape
    if weight.kind == "bf16":
        return weight.w
    out = torch.empty((n, k), dtype=torch.bfloat16, device=weight.w.device)
    stream = _lib.stream_of(out)
    if weight.kind == "int8":
        _lib.call("ltx_dequantize_w8_bf16", weight.w.data_ptr(), k, weight.scale.data_ptr(), n, k,
                  out.data_ptr(), k, stream)
    else:
        _lib.call("ltx_dequantize_mxfp8_bf16", weight.w.data_ptr(), k, weight.scale.data_ptr(), k // 32, n, k,
                  out.data_ptr(), k, stream)
    return out


_WFORMAT = {"bf16": 0, "int8": 1, "mxfp8": 2}


# Block budget of a split-K launch on explicit 128x128 tiles (tiles x splits).
SPLITK_MAX_BLOCKS = 80


@functools.lru_cache(maxsize=4096)
def auto_splits(m: int, n: int, k: int, kind: str, max_blocks: int | None = None) -> int:
    """Split-K factor of a product whose output tiles leave CUs idle, from the
    library's cost model (ltx_gemm_auto_splits); 1 when one pass is as fast.
    With ``max_blocks``, the rule for few rows on 128x128 tiles instead: the
    largest power of two that keeps at most that many blocks and at least 256
    of K per split."""
    if max_blocks is None:
        return _lib.lib().ltx_gemm_auto_splits(m, n, k, _WFORMAT.get(kind, -1))
    if m > 256 or k < 1024:
        return 1
    tiles = ((m + 127) // 128) * ((n + 127) // 128)
    if tiles >= 160:
        return 1
    unit = 128 if kind == "mxfp8" else 64
    s = 1
    while tiles * s * 2 <= max_blocks and k % (unit * s * 2) == 0 and k // (s * 2) >= 256:
        s *= 2
    return s


# Few-row products (at most ROWS_MAX_M rows: the 68 / 121-token audio stream)
# can run on the one-launch split-K kernel of ltx_gemm_rows_* with about
# ROWS_TARGET_WGS workgroups (LTX_GEMM_ROWS=1).  Off by default: inside the
# 48-block step, where these products run on the audio stream beside the
# video stream's GEMMs, its workgroups (one per CU, held for the whole K
# stream) cost the step 0.9-2.0 ms against the split-K tile kernel (two
# workgroups per CU) in A/B runs on one box, although alone it is up to 15 %
# faster on the larger audio products.
ROWS_KERNEL = os.environ.get("LTX_GEMM_ROWS", "0") == "1"
ROWS_MAX_M = int(os.environ.get("LTX_GEMM_ROWS_MAX_M", "128"))
ROWS_TARGET_WGS = int(os.environ.get("LTX_GEMM_ROWS_WGS", "256"))
_ROWS_COUNTER_WORDS = 1 << 14
_rows_counters: dict[tuple[int, int], torch.Tensor] = {}


def rows_tiles(m: int, n: int) -> int:
    """Output tiles of ltx_gemm_rows_* (its counter words): row tiles of 64, 96
    or 128 rows x column tiles of 128."""
    bm = 64 if m <= 64 else (96 if m <= 96 else 128)
    return -(-m // bm) * -(-n // 128)


def rows_splits(m: int, n: int, k: int, kind: str, target: int | None = None) -> int:
    """Split count of a few-row product: the largest power of two keeping at
    most ``target`` (default ``ROWS_TARGET_WGS``) workgroups, K divisible by
    the split granularity and at least two K stages per split."""
    target = ROWS_TARGET_WGS if target is None else target
    ks = 64 if kind == "bf16" else 128
    tiles = rows_tiles(m, n)
    s = 1
    while s < 64 and tiles * s * 2 <= target and k % (ks * s * 2) == 0 and k // (s * 2) >= 2 * ks:
        s *= 2
    return s


def rows_eligible(m: int, n: int, k: int, kind: str) -> bool:
    ks = 64 if kind == "bf16" else 128
    return ROWS_KERNEL and 0 < m <= ROWS_MAX_M and k % ks == 0 and n % 8 == 0


def _rows_counters_for(device: torch.device, stream: int, words: int) -> torch.Tensor:
    """A zeroed counter array for the calls of one stream (every call leaves
    it zero).  Cached per stream outside graph capture; under capture without
    a cached array, a fresh one whose zero fill is part of the graph."""
    key = (device.index if device.index is not None else torch.cuda.current_device(), stream)
    buf = _rows_counters.get(key)
    if buf is not None and buf.numel() >= words:
        return buf
    buf = torch.zeros(max(words, _ROWS_COUNTER_WORDS), dtype=torch.int32, device=device)
    if not torch.cuda.is_current_stream_capturing():
        _rows_counters[key] = buf
    return buf


def linear_rows(x: torch.Tensor, weight: LinearWeight, *, epilogue: int = EPI_BIAS,
                out: torch.Tensor | None = None, residual: torch.Tensor | None = None,
                gate: torch.Tensor | None = None, sigmoid_from: int | None = None,
                splits: int | None = None) -> torch.Tensor:
    """:func:`linear` for few-row x on the one-launch split-K kernel
    (ltx_gemm_rows_*): same epilogues, same rounding points."""
    k = weight.in_features
    n = weight.out_features
    if x.dtype != torch.bfloat16:
        raise TypeError(f"linear_rows expects bf16 activations, got {x.dtype}")
    xv, lda = _lib.row_view(x, k)
    m = x.numel() // k
    lead = x.shape[:-1]
    if out is None:
        out = torch.empty((*lead, n), dtype=torch.bfloat16, device=x.device)
    ov, ldc = _lib.row_view(out, n)
    if ov.data_ptr() != out.data_ptr():
        raise ValueError("out must be a row-strided view")
    rptr, ldr, gptr = None, 0, None
    if epilogue in (EPI_RESIDUAL, EPI_RESIDUAL_ROUND):
        if residual is None or gate is None:
            raise ValueError("residual epilogues need residual and gate")
        rv, ldr = _lib.row_view(residual, n)
        if rv.data_ptr() != residual.data_ptr():
            raise ValueError("residual must be a row-strided view")
        rptr = rv.data_ptr()
        gate = gate.reshape(-1).contiguous()
        if gate.dtype != torch.float32 or gate.numel() != n:
            raise ValueError("gate must be fp32 with N elements")
        gptr = gate.data_ptr()
    flags = epilogue
    if weight.qlinear and weight.bias is not None:
        flags |= _lib.GEMM_ROUND_THEN_BIAS
    sig = n if sigmoid_from is None else int(sigmoid_from)
    bptr = None if weight.bias is None else weight.bias.data_ptr()
    if m == 0:
        return out
    s = rows_splits(m, n, k, weight.kind) if splits is None else int(splits)
    stream = _lib.stream_of(x)
    ws = torch.empty(s * m * n, dtype=torch.float32, device=x.device)
    words = rows_tiles(m, n)
    cnt = _rows_counters_for(x.device, stream, words)
    args = (ws.data_ptr(), ws.numel() * 4, cnt.data_ptr(), cnt.numel(), stream)
    detail = f"rows {weight.kind} M={m} N={n} K={k} epi={epilogue} splits={s}"
    hook = LAUNCH_HOOK
    info = (weight.kind, m, n, k, epilogue)
    if hook is not None:
        hook("pre", info)
    if weight.kind == "bf16":
        _lib.call("ltx_gemm_rows_bf16", xv.data_ptr(), lda, weight.w.data_ptr(), weight.w.stride(0), bptr,
                  ov.data_ptr(), ldc, m, n, k, flags, rptr, ldr, gptr, sig, s, *args, detail=detail)
    elif weight.kind == "int8":
        _lib.call("ltx_gemm_rows_w8a16_bf16", xv.data_ptr(), lda, weight.w.data_ptr(), weight.w.stride(0),
                  weight.scale.data_ptr(), bptr, ov.data_ptr(), ldc, m, n, k, flags, rptr, ldr, gptr, sig, s,
                  *args, detail=detail)
    elif weight.kind == "mxfp8":
        _lib.call("ltx_gemm_rows_mxfp8_bf16", xv.data_ptr(), lda, weight.w.data_ptr(), weight.w.stride(0),
                  weight.scale.data_ptr(), weight.scale.stride(0), bptr, ov.data_ptr(), ldc, m, n, k, flags, rptr,
                  ldr, gptr, sig, s, *args, detail=detail)
    else:
        raise ValueError(f"unknown weight format {weight.kind!r}")
    if hook is not None:
        hook("post", info)
    return out


@dataclass
class MxRows:
    """Activation rows in MXFP8: E4M3 codes (M, K) uint8 and E8M0 scales
    (M, K/32) uint8 -- the opt-in MX path's quantised GEMM input."""

    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self):
        return self.codes.shape


def quantize_rows_mxfp8(x: torch.Tensor, codes: torch.Tensor | None = None,
                        scales: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """MXFP8 of the rows of x (..., K) bf16 with the library's encoder (the
    weights' OCP rule, blocks of 32 along K): E4M3 codes (M, K) uint8 and E8M0
    scales (M, K / 32) uint8."""
    k = x.shape[-1]
    if k % 32:
        raise ValueError(f"K={k} is not a multiple of 32")
    xv, lda = _lib.row_view(x, k)
    m = x.numel() // k
    if codes is None:
        codes = torch.empty((m, k), dtype=torch.uint8, device=x.device)
    if scales is None:
        scales = torch.empty((m, k // 32), dtype=torch.uint8, device=x.device)
    _lib.call("ltx_quantize_mxfp8_bf16", xv.data_ptr(), lda, m, k, codes.data_ptr(), codes.stride(0),
              scales.data_ptr(), scales.stride(0), _lib.stream_of(x), detail=f"activations M={m} K={k}")
    return codes, scales


def linear_mx(codes: torch.Tensor, scales: torch.Tensor, weight: LinearWeight, *, epilogue: int = EPI_BIAS,
              out: torch.Tensor | None = None, residual: torch.Tensor | None = None,
              gate: torch.Tensor | None = None, sigmoid_from: int | None = None) -> torch.Tensor:
    """``epilogue(x @ W.T + b)`` with x given as MXFP8 rows (codes (M, K),
    scales (M, K/32), from :func:`quantize_rows_mxfp8`) and MXFP8 weights, on
    the scaled fp8 MFMA; the weights' quantised-linear rounding is kept.
    Returns (M, N) bf16."""
    if weight.kind != "mxfp8":
        raise ValueError(f"linear_mx needs MXFP8 weights, got {weight.kind!r}")
    m, k = codes.shape
    n = weight.out_features
    if k != weight.in_features or scales.shape != (m, k // 32):
        raise ValueError(f"activation codes {tuple(codes.shape)} / scales {tuple(scales.shape)} do not match "
                         f"K={weight.in_features}")
    if out is None:
        out = torch.empty((m, n), dtype=torch.bfloat16, device=codes.device)
    ov, ldc = _lib.row_view(out, n)
    rptr, ldr, gptr = None, 0, None
    if epilogue in (EPI_RESIDUAL, EPI_RESIDUAL_ROUND):
        if residual is None or gate is None:
            raise ValueError("residual epilogues need residual and gate")
        rv, ldr = _lib.row_view(residual, n)
        rptr = rv.data_ptr()
        gate = gate.reshape(-1).contiguous()
        if gate.dtype != torch.float32 or gate.numel() != n:
            raise ValueError("gate must be fp32 with N elements")
        gptr = gate.data_ptr()
    flags = epilogue
    if weight.qlinear and weight.bias is not None:
        flags |= _lib.GEMM_ROUND_THEN_BIAS
    sig = n if sigmoid_from is None else int(sigmoid_from)
    bptr = None if weight.bias is None else weight.bias.data_ptr()
    _lib.call("ltx_gemm_mx_bf16", codes.data_ptr(), codes.stride(0), scales.data_ptr(), scales.stride(0),
              weight.w.data_ptr(), weight.w.stride(0), weight.scale.data_ptr(), weight.scale.stride(0), bptr,
              ov.data_ptr(), ldc, m, n, k, flags, rptr, ldr, gptr, sig, _lib.stream_of(codes),
              detail=f"mx M={m} N={n} K={k} epi={epilogue}")
    return out


def linear_mx_gelu(x: MxRows, weight: LinearWeight) -> MxRows:
    """The MX path's FF up-projection: ``mxfp8(bf16(gelu_tanh(bf16(x W^T + b))))``
    with the quantisation in the GEMM's epilogue (ltx_gemm_mx_gelu_mxfp8)."""
    if weight.kind != "mxfp8":
        raise ValueError(f"linear_mx_gelu needs MXFP8 weights, got {weight.kind!r}")
    m, k = x.codes.shape
    n = weight.out_features
    if k != weight.in_features or n % 32:
        raise ValueError(f"K={k} / N={n} do not fit the weight {weight.out_features}x{weight.in_features}")
    codes = torch.empty((m, n), dtype=torch.uint8, device=x.codes.device)
    scales = torch.empty((m, n // 32), dtype=torch.uint8, device=x.codes.device)
    flags = _lib.GEMM_ROUND_THEN_BIAS if (weight.qlinear and weight.bias is not None) else 0
    bptr = None if weight.bias is None else weight.bias.data_ptr()
    hook = LAUNCH_HOOK
    info = (weight.kind, m, n, k, EPI_GELU)
    if hook is not None:
        hook("pre", info)
    _lib.call("ltx_gemm_mx_gelu_mxfp8", x.codes.data_ptr(), x.codes.stride(0), x.scales.data_ptr(),
              x.scales.stride(0), weight.w.data_ptr(), weight.w.stride(0), weight.scale.data_ptr(),
              weight.scale.stride(0), bptr, codes.data_ptr(), n, scales.data_ptr(), n // 32, m, n, k, flags,
              _lib.stream_of(x.codes), detail=f"mx gelu M={m} N={n} K={k}")
    if hook is not None:
        hook("post", info)
    return MxRows(codes, scales)


@dataclass
class Mx4Rows:
    """Rows in MXFP4: code bytes (M, K/2) uint8 and scale words (ceil(K/128), M
    rounded up to 4) int32, as :class:`LinearWeight` holds them."""

    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self):
        return torch.Size((self.codes.shape[0], self.codes.shape[1] * 2))


def _check_mxfp4(what: str, codes: torch.Tensor, scales: torch.Tensor) -> tuple[int, int, int, int]:
    """(rows, K, code row stride, word row stride) of MXFP4 codes whose scale
    words fit them."""
    if codes.dtype is torch.uint8 and codes.dim() == 2 and scales is not None and scales.dtype is torch.int32 \
            and scales.dim() == 2:
        rows, half = codes.shape
        words, ld = scales.shape
        ldc, unit = codes.stride()
        lds, sunit = scales.stride()
        if words * 64 >= half > 0 and ld >= rows and unit == sunit == 1:
            # (the stride of an axis of one entry says nothing)
            return rows, half * 2, ldc if rows > 1 else half, lds if words > 1 else (ld + 3) // 4 * 4
    raise ValueError(f"{what}: MXFP4 operands are code bytes (rows, K/2) uint8 and scale words (ceil(K/128), >= rows) "
                     f"int32 of unit column stride, got {codes.dtype} {tuple(codes.shape)} and "
                     f"{None if scales is None else (scales.dtype, tuple(scales.shape))}")


def _whole_words(scales: torch.Tensor, rows: int, k: int, ld: int) -> tuple[torch.Tensor, int]:
    """(words, row stride) whose memory goes on to a multiple of 4 rows, as products
    read them: the given ones, or a copy."""
    end = scales.storage_offset() + (k - 1) // 128 * ld + (rows + 3) // 4 * 4
    if rows % 4 == 0 or end * 4 <= scales.untyped_storage().nbytes():
        return scales, ld
    return torch.nn.functional.pad(scales[:, :rows], (0, -rows % 4)), (rows + 3) // 4 * 4


def mxfp4_scale_words(scales: torch.Tensor) -> torch.Tensor:
    """E8M0 bytes (rows, K/32) uint8 as the scale words that MXFP4 operands
    hold: int32 (ceil(K/128), rows rounded up to 4)."""
    rows, blocks = scales.shape
    words = (blocks + 3) // 4
    out = torch.zeros((words, (rows + 3) // 4 * 4, 4), dtype=torch.uint8, device=scales.device)
    padded = torch.nn.functional.pad(scales, (0, words * 4 - blocks))
    out[:, :rows] = padded.view(rows, words, 4).transpose(0, 1)
    return out.view(torch.int32).squeeze(-1)


def mxfp4_block_scales(words: torch.Tensor, rows: int, k: int) -> torch.Tensor:
    """E8M0 bytes (rows, K/32) uint8 of scale words (:func:`mxfp4_scale_words`)."""
    b = words[:, :rows].contiguous().view(torch.uint8).view(-1, rows, 4)
    return b.transpose(0, 1).reshape(rows, -1)[:, :k // 32].contiguous()


_QUANT_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def quantize_rows_mxfp4(x: torch.Tensor) -> Mx4Rows:
    """MXFP4 of the rows of x (..., K) bf16, fp16 or fp32 (blocks of 32 along K,
    the OCP rule: X = floor(log2 max|v|) - 2, E2M1 to nearest even, saturated).
    A block with a NaN or an infinity decodes to NaN."""
    if _lib.CALLS is not None:
        where = _lib.fast_stream(x)
        rows = None if where is None else _lib.CALLS.quantize(x, *where)
        if rows is not None:
            return Mx4Rows(*_lib.launched(rows, "ltx_quantize_mxfp4"))
    k = x.shape[-1]
    dtype = _QUANT_DTYPES.get(x.dtype)
    if dtype is None:
        raise TypeError(f"quantize_rows_mxfp4 takes bf16, fp16 or fp32 rows, got {x.dtype}")
    if k % 32 or k == 0:
        raise ValueError(f"K={k} is not a positive multiple of 32")
    xv, ldx = _lib.row_view(x, k)
    m = x.numel() // k
    if m == 1:
        ldx = k  # (the stride of an axis of one entry says nothing)
    elif ldx < k:  # one row for all
        xv, ldx = xv.contiguous(), k
    ld = (m + 3) // 4 * 4
    codes = x.new_empty((m, k // 2), dtype=torch.uint8)
    scales = x.new_empty(((k + 127) // 128, ld), dtype=torch.int32)
    if m:
        st = _lib.launch(_lib.same_device(xv), "ltx_quantize_mxfp4", xv.data_ptr(), dtype, ldx, m, k,
                         codes.data_ptr(), k // 2, scales.data_ptr(), ld)
        if st:
            raise _lib.LtxKernelError("ltx_quantize_mxfp4", st, f"{x.dtype} rows M={m} K={k} ld={ldx}")
    return Mx4Rows(codes, scales)


def dequantize_rows_mxfp4(rows: Mx4Rows) -> torch.Tensor:
    """bf16 (M, K) values of MXFP4 rows, exact."""
    codes, scales = rows.codes, rows.scales
    if _lib.CALLS is not None:
        where = _lib.fast_stream(codes)
        out = None if where is None else _lib.CALLS.dequantize(codes, scales, *where)
        if out is not None:
            return _lib.launched(out, "ltx_dequantize_mxfp4_bf16")
    m, k, ldq, lds = _check_mxfp4("dequantize_rows_mxfp4", codes, scales)
    out = codes.new_empty((m, k), dtype=torch.bfloat16)
    if m:
        st = _lib.launch(_lib.same_device(codes, scales), "ltx_dequantize_mxfp4_bf16", codes.data_ptr(), ldq,
                         scales.data_ptr(), lds, m, k, out.data_ptr(), k)
        if st:
            raise _lib.LtxKernelError("ltx_dequantize_mxfp4_bf16", st, f"M={m} K={k}")
    return out


@functools.lru_cache(maxsize=4096)
def _mxfp4_workspace_bytes(name: str, m: int, n: int, k: int) -> int:
    return getattr(_lib.lib(), name)(m, n, k)


def _linear_mxfp4(x: torch.Tensor | Mx4Rows, weight: LinearWeight, epilogue: int, out: torch.Tensor | None,
                  residual: torch.Tensor | None, gate: torch.Tensor | None,
                  sigmoid_from: int | None) -> torch.Tensor:
    """:func:`linear` on MXFP4 weights, for bf16 or MXFP4 rows.  (Small products
    are bound by the host: the usual call is one native call, csrc/calls.cpp;
    this path, for all others, reads each tensor's properties once.)"""
    w, scale, bias = weight.w, weight.scale, weight.bias
    if _lib.CALLS is not None and LAUNCH_HOOK is None:
        where = _lib.fast_stream(w)
        if where is not None:
            src, xs = (x.codes, x.scales) if isinstance(x, Mx4Rows) else (x, None)
            y = _lib.CALLS.linear(src, xs, w, scale, bias,
                                  _lib.GEMM_ROUND_THEN_BIAS if weight.qlinear and bias is not None else 0, epilogue,
                                  residual, gate, -1 if sigmoid_from is None else max(int(sigmoid_from), 0), out,
                                  *where)
            if y is not None:
                return _lib.launched(y, "ltx_gemm_mxfp4_bf16" if xs is None else "ltx_gemm_mx4_bf16")
    n, k, ldw, ldws = _check_mxfp4("weight", w, scale)
    quantised = isinstance(x, Mx4Rows)
    if quantised:
        src, xs = x.codes, x.scales
        m, kx, lda, ldas = _check_mxfp4("activations", src, xs)
        xs, ldas = _whole_words(xs, m, kx, ldas)
        shape = (m, n)
    else:
        if x.dtype is not torch.bfloat16:
            raise TypeError(f"linear expects bf16 or MXFP4 activations, got {x.dtype}")
        shape, st = x.shape, x.stride()
        if len(shape) == 2 and st[1] == 1:  # rows of a matrix
            m, kx = shape
            src, lda, shape = x, st[0], (m, n)
        else:
            *lead, kx = shape
            src, lda = _lib.row_view(x, kx)
            m, shape = x.numel() // kx if kx else 0, (*lead, n)  # (K = 0 is refused below)
        if m == 1:
            lda = kx  # (the stride of an axis of one entry says nothing)
        elif lda < kx:  # one row for all
            src, lda = src.contiguous(), kx
        xs = None
    if kx != k:
        raise ValueError(f"activations have K={kx}, the weight {k}")
    given = out is not None
    if not given:
        out = src.new_empty(shape, dtype=torch.bfloat16)
        ldc = n
    else:
        if out.dtype is not torch.bfloat16 or out.shape != shape:
            raise ValueError(f"out must be bf16 {shape}, got {out.dtype} {tuple(out.shape)}")
        ov, ldc = _lib.row_view(out, n)
        if ov.data_ptr() != out.data_ptr() or (ldc < n and m > 1):
            raise ValueError("out must be a row-strided view")
        ldc = ldc if m > 1 else n
    rptr, ldr, gptr = None, 0, None
    if epilogue == EPI_RESIDUAL or epilogue == EPI_RESIDUAL_ROUND:
        if residual is None or gate is None:
            raise ValueError("residual epilogues need residual and gate")
        if residual.dtype is not torch.bfloat16 or residual.shape[-1] != n or residual.numel() != m * n:
            raise ValueError(f"residual must be bf16 ({m}, {n}), got {residual.dtype} {tuple(residual.shape)}")
        rv, ldr = _lib.row_view(residual, n)
        rptr = rv.data_ptr()
        if rptr != residual.data_ptr() or (ldr < n and m > 1):
            raise ValueError("residual must be a row-strided view")
        ldr = ldr if m > 1 else n
        if gate.dtype is not torch.float32 or gate.numel() != n:
            raise ValueError("gate must be fp32 with N elements")
        gate = _lib.flat(gate)
        gptr = gate.data_ptr()
    else:
        residual = gate = None
    flags, bptr = epilogue, None
    if bias is not None:
        if bias.dtype is not torch.float32 or bias.numel() != n or not bias.is_contiguous():
            raise ValueError(f"bias must be {n} contiguous fp32 values")
        bptr = bias.data_ptr()
        if weight.qlinear:
            flags |= _lib.GEMM_ROUND_THEN_BIAS
    if given and (any(t is not None and _lib.overlaps(out, t) for t in (src, xs, w, scale, bias, gate)) or (
            residual is not None and (out.data_ptr() != rptr or ldc != ldr) and _lib.overlaps(out, residual))):
        raise ValueError("out overlaps an operand, or the residual without being it")
    device = _lib.same_device(src, xs, w, scale, bias, out, residual, gate)
    if m == 0:
        return out
    name = "ltx_gemm_mx4_bf16" if quantised else "ltx_gemm_mxfp4_bf16"
    ws_bytes = _mxfp4_workspace_bytes("ltx_gemm_mx4_workspace_bytes" if quantised
                                      else "ltx_gemm_mxfp4_workspace_bytes", m, n, k)
    ws = src.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    hook = LAUNCH_HOOK
    info = (weight.kind, m, n, k, epilogue)
    if hook is not None:
        hook("pre", info)
    a_scale = (xs.data_ptr(), ldas) if quantised else ()
    st = _lib.launch(device, name, src.data_ptr(), lda, *a_scale, w.data_ptr(), ldw, scale.data_ptr(), ldws, bptr,
                     out.data_ptr(), ldc, m, n, k, flags, rptr, ldr, gptr,
                     n if sigmoid_from is None else int(sigmoid_from), None if ws is None else ws.data_ptr(),
                     ws_bytes)
    if st:
        raise _lib.LtxKernelError(name, st, f"M={m} N={n} K={k} epi={epilogue} lda={lda} ldw={ldw} ldc={ldc}")
    if hook is not None:
        hook("post", info)
    return out


@dataclass
class Int8Rows:
    """Activation rows in int8: codes (M, K) int8 and fp32 scales (M); a row's
    values are its codes times its scale."""

    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self):
        return self.codes.shape


def _check_int8(what: str, codes: torch.Tensor, scales: torch.Tensor | None) -> tuple[int, int, int]:
    """(rows, K, code row stride) of int8 codes with a scale for each row."""
    if codes.dtype is torch.int8 and codes.dim() == 2 and scales is not None and scales.dtype is torch.float32 \
            and scales.dim() == 1 and scales.is_contiguous():
        rows, k = codes.shape
        ld, unit = codes.stride()
        if k > 0 and scales.shape[0] == rows and unit == 1 and (rows <= 1 or ld >= k):
            return rows, k, ld if rows > 1 else (k + 15) // 16 * 16  # (the stride of an axis of one entry says nothing)
    raise ValueError(f"{what}: int8 operands are codes (rows, K) int8 of unit column stride and contiguous fp32 scales "
                     f"(rows), got {codes.dtype} {tuple(codes.shape)} and "
                     f"{None if scales is None else (scales.dtype, tuple(scales.shape))}")


def quantize_rows_int8(x: torch.Tensor) -> Int8Rows:
    """int8 of the rows of x (..., K) bf16, fp16 or fp32 by the int8 weights' rule:
    scale = max|v| / 127, codes v / scale to the nearest, ties to even (both
    quotients in fp32).  A row of zeros has scale 0; one with a NaN or an infinity
    scale NaN, which its products and its decoded values take."""
    if _lib.CALLS is not None:
        where = _lib.fast_stream(x)
        rows = None if where is None else _lib.CALLS.quantize8(x, *where)
        if rows is not None:
            return Int8Rows(*_lib.launched(rows, "ltx_quantize_int8"))
    k = x.shape[-1]
    dtype = _QUANT_DTYPES.get(x.dtype)
    if dtype is None:
        raise TypeError(f"quantize_rows_int8 takes bf16, fp16 or fp32 rows, got {x.dtype}")
    if k % 16 or k == 0:
        raise ValueError(f"K={k} is not a positive multiple of 16")
    xv, ldx = _lib.row_view(x, k)
    m = x.numel() // k
    if m == 1:
        ldx = k  # (the stride of an axis of one entry says nothing)
    elif ldx < k:  # one row for all
        xv, ldx = xv.contiguous(), k
    codes = x.new_empty((m, k), dtype=torch.int8)
    scales = x.new_empty(m, dtype=torch.float32)
    if m:
        st = _lib.launch(_lib.same_device(xv), "ltx_quantize_int8", xv.data_ptr(), dtype, ldx, m, k, codes.data_ptr(), k,
                         scales.data_ptr())
        if st:
            raise _lib.LtxKernelError("ltx_quantize_int8", st, f"{x.dtype} rows M={m} K={k} ld={ldx}")
    return Int8Rows(codes, scales)


def dequantize_rows_int8(rows: Int8Rows) -> torch.Tensor:
    """bf16 (M, K) values of int8 rows: codes times scales, rounded once."""
    codes, scales = rows.codes, rows.scales
    if _lib.CALLS is not None:
        where = _lib.fast_stream(codes)
        out = None if where is None else _lib.CALLS.dequantize8(codes, scales, *where)
        if out is not None:
            return _lib.launched(out, "ltx_dequantize_w8_bf16")
    m, k, ldq = _check_int8("dequantize_rows_int8", codes, scales)
    out = codes.new_empty((m, k), dtype=torch.bfloat16)
    if m:
        st = _lib.launch(_lib.same_device(codes, scales), "ltx_dequantize_w8_bf16", codes.data_ptr(), ldq,
                         scales.data_ptr(), m, k, out.data_ptr(), k)
        if st:
            raise _lib.LtxKernelError("ltx_dequantize_w8_bf16", st, f"M={m} K={k}")
    return out


@functools.lru_cache(maxsize=4096)
def _int8_workspace_bytes(m: int, n: int, k: int) -> int:
    return _lib.lib().ltx_gemm_i8_workspace_bytes(m, n, k)


def _linear_int8(x: Int8Rows, weight: LinearWeight, epilogue: int, out: torch.Tensor | None,
                 residual: torch.Tensor | None, gate: torch.Tensor | None, sigmoid_from: int | None,
                 watched: bool = False) -> torch.Tensor:
    """:func:`linear` for int8 rows and int8 weights (``watched``: inside its caller's calls of the launch observer)."""
    w, scale, bias = weight.w, weight.scale, weight.bias
    codes, xs = x.codes, x.scales
    hook = None if watched else LAUNCH_HOOK
    if _lib.CALLS is not None and hook is None:
        where = _lib.fast_stream(w)
        if where is not None:
            y = _lib.CALLS.linear8(codes, xs, w, scale, bias,
                                   _lib.GEMM_ROUND_THEN_BIAS if weight.qlinear and bias is not None else 0, epilogue,
                                   residual, gate, -1 if sigmoid_from is None else max(int(sigmoid_from), 0), out,
                                   *where)
            if y is not None:
                return _lib.launched(y, "ltx_gemm_i8_bf16")
    n, k, ldw = _check_int8("weight", w, scale)
    m, kx, lda = _check_int8("activations", codes, xs)
    if kx != k:
        raise ValueError(f"activations have K={kx}, the weight {k}")
    given = out is not None
    if not given:
        out = codes.new_empty((m, n), dtype=torch.bfloat16)
        ldc = n
    else:
        if out.dtype is not torch.bfloat16 or out.shape != (m, n):
            raise ValueError(f"out must be bf16 {(m, n)}, got {out.dtype} {tuple(out.shape)}")
        ov, ldc = _lib.row_view(out, n)
        if ov.data_ptr() != out.data_ptr() or (ldc < n and m > 1):
            raise ValueError("out must be a row-strided view")
        ldc = ldc if m > 1 else n
    rptr, ldr, gptr = None, 0, None
    if epilogue == EPI_RESIDUAL or epilogue == EPI_RESIDUAL_ROUND:
        if residual is None or gate is None:
            raise ValueError("residual epilogues need residual and gate")
        if residual.dtype is not torch.bfloat16 or residual.shape[-1] != n or residual.numel() != m * n:
            raise ValueError(f"residual must be bf16 ({m}, {n}), got {residual.dtype} {tuple(residual.shape)}")
        rv, ldr = _lib.row_view(residual, n)
        rptr = rv.data_ptr()
        if rptr != residual.data_ptr() or (ldr < n and m > 1):
            raise ValueError("residual must be a row-strided view")
        ldr = ldr if m > 1 else n
        if gate.dtype is not torch.float32 or gate.numel() != n:
            raise ValueError("gate must be fp32 with N elements")
        gate = _lib.flat(gate)
        gptr = gate.data_ptr()
    else:
        residual = gate = None
    flags, bptr = epilogue, None
    if bias is not None:
        if bias.dtype is not torch.float32 or bias.numel() != n or not bias.is_contiguous():
            raise ValueError(f"bias must be {n} contiguous fp32 values")
        bptr = bias.data_ptr()
        if weight.qlinear:
            flags |= _lib.GEMM_ROUND_THEN_BIAS
    if given and (any(t is not None and _lib.overlaps(out, t) for t in (codes, xs, w, scale, bias, gate)) or (
            residual is not None and (out.data_ptr() != rptr or ldc != ldr) and _lib.overlaps(out, residual))):
        raise ValueError("out overlaps an operand, or the residual without being it")
    device = _lib.same_device(codes, xs, w, scale, bias, out, residual, gate)
    if m == 0:
        return out
    ws_bytes = _int8_workspace_bytes(m, n, k)
    ws = codes.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    info = ("w8a8", m, n, k, epilogue)
    if hook is not None:
        hook("pre", info)
    st = _lib.launch(device, "ltx_gemm_i8_bf16", codes.data_ptr(), lda, xs.data_ptr(), w.data_ptr(), ldw,
                     scale.data_ptr(), bptr, out.data_ptr(), ldc, m, n, k, flags, rptr, ldr, gptr,
                     n if sigmoid_from is None else int(sigmoid_from), None if ws is None else ws.data_ptr(), ws_bytes)
    if st:
        raise _lib.LtxKernelError("ltx_gemm_i8_bf16", st, f"M={m} N={n} K={k} epi={epilogue} lda={lda} ldw={ldw} "
                                                         f"ldc={ldc}")
    if hook is not None:
        hook("post", info)
    return out


def _mx_eligible(m: int, n: int, k: int, weight: LinearWeight, tile: int) -> bool:
    return (MX_ACTIVATIONS and weight.kind == "mxfp8" and tile in (TILE_AUTO, TILE_G8) and k % 512 == 0
            and ((m + 255) // 256) * ((n + 255) // 256) >= MX_MIN_TILES)


def _int8_eligible(x, weight: LinearWeight, tile: int, splits: int | None) -> bool:
    return (INT8_ACTIVATIONS and weight.kind == "int8" and tile in (TILE_AUTO, TILE_G8) and splits is None
            and isinstance(x, torch.Tensor) and x.dtype is torch.bfloat16 and weight.in_features % 64 == 0
            and weight.in_features < 1 << 17)


def _linear_int8_rows(x: torch.Tensor, weight: LinearWeight, epilogue: int, out: torch.Tensor | None,
                      residual: torch.Tensor | None, gate: torch.Tensor | None,
                      sigmoid_from: int | None) -> torch.Tensor:
    """:func:`linear` of bf16 rows (..., K) through int8 rows."""
    lead, n = x.shape[:-1], weight.out_features
    hook = LAUNCH_HOOK if x.numel() else None
    info = ("w8a8", x.numel() // max(x.shape[-1], 1), n, weight.in_features, epilogue)
    if hook is not None:
        hook("pre", info)
    rows = quantize_rows_int8(x)
    rest = residual, gate, sigmoid_from, hook is not None
    if len(lead) == 1 or out is None:
        y = _linear_int8(rows, weight, epilogue, out, *rest)
        y = y if len(lead) == 1 else y.view(*lead, n)
    else:
        if out.shape != (*lead, n):
            raise ValueError(f"out must have the shape {(*lead, n)}, got {tuple(out.shape)}")
        ov, ldc = _lib.row_view(out, n)
        if ov.data_ptr() != out.data_ptr():
            raise ValueError("out must be a row-strided view")
        _linear_int8(rows, weight, epilogue, out.as_strided((rows.codes.shape[0], n), (ldc, 1)), *rest)
        y = out
    if hook is not None:
        hook("post", info)
    return y


def rowss_eligible(x: torch.Tensor, weight: LinearWeight) -> bool:
    """Whether :func:`linear_rowss` takes this product: bf16 activations,
    weights of one of the three formats, at least 100 tiles of 256x256 (where
    the automatic choice is the 8-wave or the mid-size kernel, whose epilogues
    give the statistics, and the same one for :func:`linear`) and the 8-wave
    kernel's conditions (MXFP8 weights: K a multiple of 512), outside the
    opt-in MX and int8 paths.  Not bf16 products of 160 tiles on with fewer columns than
    K (the A2V query projection of long clips): the attention with its norm
    inside measured slower than with the separate pass (6144 x 68 tokens 144
    against 138 us, 14640 x 68 324 against 316)."""
    if isinstance(x, MxRows) or x.dtype != torch.bfloat16 or weight.kind not in ("bf16", "int8", "mxfp8"):
        return False
    k, n = weight.in_features, weight.out_features
    m = x.numel() // max(k, 1)
    tiles = ((m + 255) // 256) * ((n + 255) // 256)
    if tiles < 100 or (weight.kind == "bf16" and tiles >= 160 and n < k):
        return False
    if weight.kind == "mxfp8" and (k % 512 or _mx_eligible(m, n, k, weight, TILE_AUTO)):
        return False
    if _int8_eligible(x, weight, TILE_AUTO, None):
        return False
    return True


def single_g8_round(x: torch.Tensor, weight: LinearWeight) -> bool:
    """Whether the product is one partial round of the 8-wave kernel (100-159
    tiles of 256x256), where the automatic choice may be the mid-size kernel."""
    if not rowss_eligible(x, weight):
        return False
    m = x.numel() // weight.in_features
    return ((m + 255) // 256) * ((weight.out_features + 255) // 256) < 160


def linear_rowss(x: torch.Tensor, weight: LinearWeight, ss_cols: int, *, sigmoid_from: int | None = None,
                 tile: int = TILE_AUTO) -> tuple[torch.Tensor, torch.Tensor]:
    """:func:`linear` with the bias epilogue on the mid-size or the 8-wave
    kernel (the automatic choice, or ``tile``), plus the per-row sums of squares of the bf16 outputs of columns [0, ss_cols) in
    fp32 partials of 64 columns: returns (out (M, N) bf16, ss (M, ss_cols/64)
    fp32) (ltx_gemm_rowss_bf16).  ``out`` is bit-identical to :func:`linear`
    with the same ``tile`` (and one split)."""
    k = weight.in_features
    n = weight.out_features
    if not rowss_eligible(x, weight):
        raise ValueError(f"linear_rowss does not take {weight.kind} weights / {x.dtype} activations here")
    xv, lda = _lib.row_view(x, k)
    m = x.numel() // k
    out = torch.empty((m, n), dtype=torch.bfloat16, device=x.device)
    parts = ss_cols // 64
    ss = torch.empty((m, parts), dtype=torch.float32, device=x.device)
    flags = EPI_BIAS | (tile << 8)
    if weight.qlinear and weight.bias is not None:
        flags |= _lib.GEMM_ROUND_THEN_BIAS
    sig = n if sigmoid_from is None else int(sigmoid_from)
    bptr = None if weight.bias is None else weight.bias.data_ptr()
    fmt = _WFORMAT[weight.kind]
    sptr, lds = (None, 0) if weight.kind == "bf16" else (
        weight.scale.data_ptr(), weight.scale.stride(0) if weight.kind == "mxfp8" else 0)
    hook = LAUNCH_HOOK
    info = (weight.kind, m, n, k, EPI_BIAS) if hook is not None else None
    if hook is not None:
        hook("pre", info)
    if m > 0:
        _lib.call("ltx_gemm_rowss_bf16", fmt, xv.data_ptr(), lda, weight.w.data_ptr(), weight.w.stride(0), sptr,
                  lds, bptr, out.data_ptr(), n, m, n, k, flags, sig, ss.data_ptr(), parts, ss_cols,
                  _lib.stream_of(x), detail=f"rowss {weight.kind} M={m} N={n} K={k} ss_cols={ss_cols}")
    if hook is not None:
        hook("post", info)
    return out, ss


def linear(x: torch.Tensor | MxRows | Mx4Rows | Int8Rows, weight: LinearWeight, *, epilogue: int = EPI_BIAS,
           out: torch.Tensor | None = None, residual: torch.Tensor | None = None,
           gate: torch.Tensor | None = None, tile: int = TILE_AUTO,
           sigmoid_from: int | None = None, splits: int | None = None) -> torch.Tensor:
    """``epilogue(x @ W.T + b)`` for x (..., K) bf16; returns (..., N) bf16.

    For the residual epilogues, ``residual`` (..., N) bf16 and ``gate`` fp32
    (N) are required; ``out`` may be ``residual`` itself (in-place update);
    on MXFP4 weights anything else that it shares with an operand is refused.
    With ``EPI_BIAS``, columns ``n >= sigmoid_from`` get the 2*sigmoid head
    gate instead (fused gate-logit columns of a Q/QKV projection).
    ``splits``: split-K factor (None: ``auto_splits`` with the automatic tile
    choice and for the 128x128 tiles, 1: single pass); the split form sums fp32
    partials from a workspace.
    With ``ROWS_KERNEL`` set, few-row products with ``splits=None`` and the
    automatic tile choice run on :func:`linear_rows`.
    MXFP4 weights take bf16 rows or :class:`Mx4Rows` and choose tiles and
    splits themselves (``tile`` and ``splits`` stay at their defaults); so do
    int8 weights with :class:`Int8Rows`, which refuse the same outputs.
    """
    if isinstance(x, Int8Rows):
        if weight.kind != "int8":
            raise ValueError(f"Int8Rows activations do not go with {weight.kind} weights")
        if tile != TILE_AUTO or splits is not None:
            raise ValueError("products of int8 rows take no explicit tile or split count")
        return _linear_int8(x, weight, epilogue, out, residual, gate, sigmoid_from)
    if weight.kind == "mxfp4" or isinstance(x, Mx4Rows):
        if weight.kind != "mxfp4" or isinstance(x, MxRows):
            raise ValueError(f"{type(x).__name__} activations do not go with {weight.kind} weights")
        if tile != TILE_AUTO or splits is not None:
            raise ValueError("MXFP4 products take no explicit tile or split count")
        return _linear_mxfp4(x, weight, epilogue, out, residual, gate, sigmoid_from)
    if _int8_eligible(x, weight, tile, splits):
        return _linear_int8_rows(x, weight, epilogue, out, residual, gate, sigmoid_from)
    k = weight.in_features
    n = weight.out_features
    if (splits is None and tile == TILE_AUTO and not isinstance(x, MxRows)
            and rows_eligible(x.numel() // max(k, 1), n, k, weight.kind)):
        return linear_rows(x, weight, epilogue=epilogue, out=out, residual=residual, gate=gate,
                           sigmoid_from=sigmoid_from)
    if isinstance(x, MxRows):  # quantised rows of the opt-in MX path
        hook = LAUNCH_HOOK
        info = (weight.kind, x.codes.shape[0], n, k, epilogue)
        if hook is not None:
            hook("pre", info)
        out = linear_mx(x.codes, x.scales, weight, epilogue=epilogue, out=out, residual=residual, gate=gate,
                        sigmoid_from=sigmoid_from)
        if hook is not None:
            hook("post", info)
        return out
    if x.dtype != torch.bfloat16:
        raise TypeError(f"linear expects bf16 activations, got {x.dtype}")
    xv, lda = _lib.row_view(x, k)
    m = x.numel() // k
    lead = x.shape[:-1]
    if out is None:
        out = torch.empty((*lead, n), dtype=torch.bfloat16, device=x.device)
    ov, ldc = _lib.row_view(out, n)
    if ov.data_ptr() != out.data_ptr():
        raise ValueError("out must be a row-strided view")
    rptr, ldr, gptr = None, 0, None
    if epilogue in (EPI_RESIDUAL, EPI_RESIDUAL_ROUND):
        if residual is None or gate is None:
            raise ValueError("residual epilogues need residual and gate")
        rv, ldr = _lib.row_view(residual, n)
        if rv.data_ptr() != residual.data_ptr():
            raise ValueError("residual must be a row-strided view")
        rptr = rv.data_ptr()
        if gate.dtype != torch.float32 or gate.numel() != n:
            raise ValueError("gate must be fp32 with N elements")
        gate = _lib.flat(gate)
        gptr = gate.data_ptr()
    flags = epilogue | (tile << 8)
    if weight.qlinear and weight.bias is not None:
        flags |= _lib.GEMM_ROUND_THEN_BIAS
    sig = n if sigmoid_from is None else int(sigmoid_from)
    bias = weight.bias
    bptr = None if bias is None else bias.data_ptr()
    stream = _lib.stream_of(x)
    detail = f"{weight.kind} M={m} N={n} K={k} epi={epilogue}"
    hook = LAUNCH_HOOK
    info = (weight.kind, m, n, k, epilogue) if hook is not None else None
    if splits is None:
        splits = (auto_splits(m, n, k, weight.kind) if tile == TILE_AUTO else
                  auto_splits(m, n, k, weight.kind, SPLITK_MAX_BLOCKS) if tile == TILE_128 else 1)
    if hook is not None:
        hook("pre", info)
    if splits == 1 and _mx_eligible(m, n, k, weight, tile):
        codes, scales = quantize_rows_mxfp8(x)
        linear_mx(codes, scales, weight, epilogue=epilogue, out=ov, residual=residual, gate=gate,
                  sigmoid_from=sigmoid_from)
        if hook is not None:
            hook("post", info)
        return out
    if splits > 1:
        ws_bytes = splits * m * n * 4
        ws = torch.empty(splits * m * n, dtype=torch.float32, device=x.device)
        if weight.kind == "bf16":
            _lib.call("ltx_gemm_splitk_bf16", xv.data_ptr(), lda, weight.w.data_ptr(), weight.w.stride(0), bptr,
                      ov.data_ptr(), ldc, m, n, k, flags, rptr, ldr, gptr, sig, splits, ws.data_ptr(), ws_bytes,
                      stream, detail=detail)
        elif weight.kind == "int8":
            _lib.call("ltx_gemm_splitk_w8a16_bf16", xv.data_ptr(), lda, weight.w.data_ptr(), weight.w.stride(0),
                      weight.scale.data_ptr(), bptr, ov.data_ptr(), ldc, m, n, k, flags, rptr, ldr, gptr, sig,
                      splits, ws.data_ptr(), ws_bytes, stream, detail=detail)
        elif weight.kind == "mxfp8":
            _lib.call("ltx_gemm_splitk_mxfp8_bf16", xv.data_ptr(), lda, weight.w.data_ptr(), weight.w.stride(0),
                      weight.scale.data_ptr(), weight.scale.stride(0), bptr, ov.data_ptr(), ldc, m, n, k, flags,
                      rptr, ldr, gptr, sig, splits, ws.data_ptr(), ws_bytes, stream, detail=detail)
        else:
            raise ValueError(f"unknown weight format {weight.kind!r}")
        if hook is not None:
            hook("post", info)
        return out
    if weight.kind == "bf16":
        _lib.call("ltx_gemm_bf16", xv.data_ptr(), lda, weight.w.data_ptr(), weight.w.stride(0), bptr,
                  ov.data_ptr(), ldc, m, n, k, flags, rptr, ldr, gptr, sig, stream, detail=detail)
    elif weight.kind == "int8":
        _lib.call("ltx_gemm_w8a16_bf16", xv.data_ptr(), lda, weight.w.data_ptr(), weight.w.stride(0),
                  weight.scale.data_ptr(), bptr, ov.data_ptr(), ldc, m, n, k, flags, rptr, ldr, gptr, sig, stream,
                  detail=detail)
    elif weight.kind == "mxfp8":
        _lib.call("ltx_gemm_mxfp8_bf16", xv.data_ptr(), lda, weight.w.data_ptr(), weight.w.stride(0),
                  weight.scale.data_ptr(), weight.scale.stride(0), bptr, ov.data_ptr(), ldc, m, n, k, flags,
                  rptr, ldr, gptr, sig, stream, detail=detail)
    else:
        raise ValueError(f"unknown weight format {weight.kind!r}")
    if hook is not None:
        hook("post", info)
    return out
