"""ctypes binding of libltx_hip.so (declarations mirror include/ltx_hip.h).

The library is loaded lazily on first use.  A missing or unloadable library
raises immediately: there is no silent CPU or eager fallback behind these
entry points.
"""

from __future__ import annotations

import ctypes
import importlib.util
import os
import sys
import warnings
from pathlib import Path

import torch

LIB_NAME = "libltx_hip.so"
LIB_PATH = Path(os.environ.get("LTX_HIP_LIB", Path(__file__).with_name(LIB_NAME)))

_i64 = ctypes.c_int64
_int = ctypes.c_int
_f32 = ctypes.c_float
_f64 = ctypes.c_double
_vp = ctypes.c_void_p

# name -> argtypes (functions return int: a status, or for
# ltx_gemm_auto_splits / _rows the choice; those of SIZES an int64)
SIGNATURES: dict[str, list] = {
    "ltx_version": [],
    "ltx_device_clock_stamp": [_vp, _vp],
    "ltx_adaln_norm_fused_bf16": [_vp, _i64, _vp, _vp, _vp, _i64, _i64, _i64, _f32, _int, _vp],
    "ltx_gated_add_fused_bf16": [_vp, _i64, _vp, _i64, _vp, _vp, _i64, _i64, _i64, _int, _vp],
    "ltx_qknorm_rope_bf16": [
        _vp, _i64, _i64, _vp, _vp, _vp,
        _vp, _i64, _i64, _vp, _vp, _vp,
        _i64, _i64, _f32, _vp,
    ],
    "ltx_output_norm_modulate_bf16": [_vp, _i64, _vp, _vp, _vp, _i64, _i64, _i64, _f32, _vp],
    "ltx_euler_x0_step_bf16": [_vp, _vp, _f32, _f32, _vp, _i64, _vp],
    "ltx_timestep_embedding_f32": [_vp, _i64, _f32, _vp, _i64, _vp],
    "ltx_adaln_mlps_f32": [_vp, _i64, _vp],
    "ltx_gemv_f32_bf16w": [_vp, _i64, _i64, _vp, _vp, _vp, _i64, _int, _vp],
    "ltx_gemm_bf16": [_vp, _i64, _vp, _i64, _vp, _vp, _i64, _i64, _i64, _i64, _int, _vp, _i64, _vp, _i64, _vp],
    "ltx_gemm_w8a16_bf16": [_vp, _i64, _vp, _i64, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _int, _vp, _i64, _vp,
                            _i64, _vp],
    "ltx_gemm_mxfp8_bf16": [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _i64, _i64, _i64, _i64, _int, _vp, _i64,
                            _vp, _i64, _vp],
    "ltx_gemm_rowss_bf16": [_int, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _i64, _i64, _i64, _i64, _int, _i64,
                            _vp, _i64, _i64, _vp],
    "ltx_gemm_auto_splits": [_i64, _i64, _i64, _int],
    "ltx_gemm_auto_rows": [_i64, _i64, _i64, _int, _int],
    "ltx_gemm_splitk_bf16": [_vp, _i64, _vp, _i64, _vp, _vp, _i64, _i64, _i64, _i64, _int, _vp, _i64, _vp, _i64,
                             _int, _vp, _i64, _vp],
    "ltx_gemm_splitk_w8a16_bf16": [_vp, _i64, _vp, _i64, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _int, _vp, _i64,
                                   _vp, _i64, _int, _vp, _i64, _vp],
    "ltx_gemm_splitk_mxfp8_bf16": [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _i64, _i64, _i64, _i64, _int, _vp,
                                   _i64, _vp, _i64, _int, _vp, _i64, _vp],
    "ltx_gemm_rows_bf16": [_vp, _i64, _vp, _i64, _vp, _vp, _i64, _i64, _i64, _i64, _int, _vp, _i64, _vp, _i64,
                           _int, _vp, _i64, _vp, _i64, _vp],
    "ltx_gemm_rows_w8a16_bf16": [_vp, _i64, _vp, _i64, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _int, _vp, _i64,
                                 _vp, _i64, _int, _vp, _i64, _vp, _i64, _vp],
    "ltx_gemm_rows_mxfp8_bf16": [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _i64, _i64, _i64, _i64, _int, _vp,
                                 _i64, _vp, _i64, _int, _vp, _i64, _vp, _i64, _vp],
    "ltx_gemm_mx_bf16": [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _i64, _i64, _i64, _i64, _int, _vp,
                         _i64, _vp, _i64, _vp],
    "ltx_gemm_mx_gelu_mxfp8": [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _i64, _vp, _i64, _i64, _i64,
                               _i64, _int, _vp],
    "ltx_quantize_mxfp8_bf16": [_vp, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp],
    "ltx_dequantize_mxfp8_bf16": [_vp, _i64, _vp, _i64, _i64, _i64, _vp, _i64, _vp],
    "ltx_quantize_w8_bf16": [_vp, _i64, _i64, _i64, _vp, _i64, _vp, _vp],
    "ltx_dequantize_w8_bf16": [_vp, _i64, _vp, _i64, _i64, _vp, _i64, _vp],
    "ltx_gemm_mxfp4_workspace_bytes": [_i64, _i64, _i64],
    "ltx_gemm_mx4_workspace_bytes": [_i64, _i64, _i64],
    "ltx_gemm_mxfp4_bf16": [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _i64, _i64, _i64, _i64, _int, _vp, _i64, _vp,
                            _i64, _vp, _i64, _vp],
    "ltx_gemm_mx4_bf16": [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _i64, _i64, _i64, _i64, _int, _vp,
                          _i64, _vp, _i64, _vp, _i64, _vp],
    "ltx_quantize_mxfp4": [_vp, _int, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp],
    "ltx_dequantize_mxfp4_bf16": [_vp, _i64, _vp, _i64, _i64, _i64, _vp, _i64, _vp],
    "ltx_rotary": [_vp, _vp, _int, _i64, _i64, _i64, _i64, _vp, _int, _i64, _vp, _f64, _int, _vp],
    "ltx_headnorm_rotary": [_vp, _vp, _int, _i64, _i64, _i64, _i64, _vp, _int, _i64, _vp, _f64, _f64, _f64, _int, _vp],
    "ltx_headnorm_rotary_grad_workspace_bytes": [_i64],
    "ltx_headnorm_rotary_grad": [_vp, _vp, _int, _i64, _i64, _i64, _i64, _vp, _int, _i64, _vp, _f64, _f64, _f64, _int,
                                 _vp, _i64, _vp],
    "ltx_quantize_int8": [_vp, _int, _i64, _i64, _i64, _vp, _i64, _vp, _vp],
    "ltx_gemm_i8_workspace_bytes": [_i64, _i64, _i64],
    "ltx_gemm_i8_bf16": [_vp, _i64, _vp, _vp, _i64, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _int, _vp, _i64, _vp, _i64,
                         _vp, _i64, _vp],
    "ltx_dequantize_fp8_e4m3": [_vp, _i64, _vp, _vp, _int, _vp],
    "ltx_attn_transpose_v_bf16": [_vp, _i64, _i64, _i64, _i64, _vp, _i64, _vp],
    "ltx_flash_attn_bf16": [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _i64, _f32, _vp],
    "ltx_flash_attn_splitkv_bf16": [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _i64,
                                    _f32, _i64, _vp, _i64, _vp],
    "ltx_flash_attn_splitkv_noalloc_bf16": [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64,
                                            _i64, _i64, _f32, _i64, _vp],
    "ltx_adaln_norm_fused2_bf16": [_vp, _i64, _vp, _vp, _vp, _i64, _vp, _vp, _vp, _i64, _i64, _i64, _f32, _int,
                                   _vp],
    "ltx_qknorm_rope_axes_bf16": [_vp, _i64, _i64, _vp, _vp, _vp, _vp, _i64, _i64, _vp, _i64, _i64, _vp, _vp, _vp,
                                  _vp, _i64, _i64, _i64, _i64, _f32, _vp],
    "ltx_flash_attn_v_bf16": [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _i64, _f32,
                              _vp],
    "ltx_flash_attn_qnorm_v_bf16": [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64,
                                    _i64, _f32, _vp, _i64, _i64, _vp, _f32, _vp, _vp, _vp, _i64, _i64, _vp],
    "ltx_flash_attn_splitkv_v_bf16": [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64,
                                      _i64, _f32, _i64, _vp, _i64, _vp],
    "ltx_broadcast_add_f32": [_vp, _vp, _vp, _i64, _i64, _vp],
    "ltx_x0_from_velocity_f32": [_vp, _vp, _f32, _vp, _i64, _vp],
    "ltx_guidance_f32": [_vp, _vp, _vp, _vp, _f32, _f32, _f32, _vp, _vp, _vp, _i64, _int, _vp],
    "ltx_guidance_stats_f32": [_vp, _vp, _i64, _int, _f32, _f32, _vp, _vp],
    "ltx_ge_correct_f32": [_vp, _vp, _vp, _int, _f32, _f32, _i64, _vp],
    "ltx_euler_step_bf16": [_vp, _vp, _f32, _vp, _i64, _vp],
    "ltx_swap_axes": [_vp, _i64, _i64, _i64, _int, _vp, _vp],
    "ltx_gemma_features_bf16": [_vp, _i64, _i64, _i64, _i64, _i64, _vp, _f32, _f32, _f32, _vp, _vp, _i64, _vp],
}

# Functions of SIGNATURES whose result is a size (int64)
SIZES = ("ltx_gemm_mxfp4_workspace_bytes", "ltx_gemm_mx4_workspace_bytes", "ltx_gemm_i8_workspace_bytes",
         "ltx_headnorm_rotary_grad_workspace_bytes")


class RotaryRows(ctypes.Structure):
    """``ltx_rotary_rows``: a tensor and where its result goes."""

    _fields_ = [("x", _vp), ("x_batch", _i64), ("x_token", _i64), ("x_head", _i64),
                ("out", _vp), ("out_batch", _i64), ("out_token", _i64), ("out_head", _i64), ("heads", _i64)]


class HeadnormRows(ctypes.Structure):
    """``ltx_headnorm_rows``: a tensor, where its result goes, the gradient of the
    forward result, the norm weights and where their gradient goes."""

    _fields_ = [("x", _vp), ("x_batch", _i64), ("x_token", _i64), ("x_head", _i64),
                ("out", _vp), ("out_batch", _i64), ("out_token", _i64), ("out_head", _i64),
                ("g", _vp), ("g_batch", _i64), ("g_token", _i64), ("g_head", _i64),
                ("weight", _vp), ("dweight", _vp), ("heads", _i64)]


# Flag values (include/ltx_hip.h)
ADALN_ROUND_NORM = 1
ADALN_NO_NORM = 2
GATED_ROUND_PRODUCT = 1
GEMV_SILU_INPUT = 1
GEMV_SILU_OUTPUT = 2
GEMM_EPI_BIAS = 0
GEMM_EPI_GELU = 1
GEMM_EPI_RESIDUAL = 2
GEMM_EPI_RESIDUAL_ROUND = 3
GEMM_EPI_SIGMOID2 = 4
GEMM_TILE_256 = 1 << 8
GEMM_TILE_128 = 2 << 8
GEMM_TILE_256_DMA = 3 << 8
GEMM_TILE_256x128 = 4 << 8
GEMM_TILE_G8 = 5 << 8
GEMM_TILE_G8_128 = 6 << 8
GEMM_ROUND_THEN_BIAS = 1 << 12
ROTARY_INTERLEAVED = 1
ROTARY_TRANSPOSE = 2
# Status of a request above the fixed scratch of a no-allocation entry point
ERR_SCRATCH_LIMIT = -5
ATTN_NOALLOC_SCRATCH_BYTES = 32 << 20

_LIB: ctypes.CDLL | None = None
# Native host side of the small MXFP4, int8, rotary and per-head norm calls (csrc/calls.cpp,
# the _calls.so beside the library), once that is loaded; None where there is none for this Python and
# torch: their Python path does the same
CALLS = None
_CALLS_ENTRIES = ("ltx_gemm_mxfp4_bf16", "ltx_gemm_mxfp4_workspace_bytes", "ltx_gemm_mx4_bf16",
                  "ltx_gemm_mx4_workspace_bytes", "ltx_quantize_mxfp4", "ltx_dequantize_mxfp4_bf16", "ltx_rotary",
                  "ltx_quantize_int8", "ltx_dequantize_w8_bf16", "ltx_gemm_i8_bf16", "ltx_gemm_i8_workspace_bytes",
                  "ltx_headnorm_rotary", "ltx_headnorm_rotary_grad", "ltx_headnorm_rotary_grad_workspace_bytes")
_current_device = getattr(torch._C, "_cuda_getDevice", None)  # (None: a torch without a GPU backend)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def lib() -> ctypes.CDLL:
    """Return the loaded library, loading it on first call."""
    global _LIB, CALLS
    if _LIB is None:
        if not LIB_PATH.exists():
            raise RuntimeError(
                f"{LIB_PATH} is not built; run `python ltx-2-mlx_amd/build_lib.py` "
                "(or __graft_entry__.build())"
            )
        handle = ctypes.CDLL(str(LIB_PATH))
        for name, argtypes in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.argtypes = argtypes
            fn.restype = ctypes.c_int
        for name in SIZES:
            getattr(handle, name).restype = _i64
        handle.ltx_attn_vt_padded_len.argtypes = [_i64]
        handle.ltx_attn_vt_padded_len.restype = _i64
        handle.ltx_attn_splitkv_workspace_bytes.argtypes = [_i64, _i64, _i64, _i64]
        handle.ltx_attn_splitkv_workspace_bytes.restype = _i64
        handle.ltx_gemm_splitk_workspace_bytes.argtypes = [_i64, _i64, _i64]
        handle.ltx_gemm_splitk_workspace_bytes.restype = _i64
        handle.ltx_gemm_rows_workspace_bytes.argtypes = [_i64, _i64, _i64]
        handle.ltx_gemm_rows_workspace_bytes.restype = _i64
        handle.ltx_gemm_rows_counter_words.argtypes = [_i64, _i64]
        handle.ltx_gemm_rows_counter_words.restype = _i64
        handle.ltx_status_string.argtypes = [ctypes.c_int]
        handle.ltx_status_string.restype = ctypes.c_char_p
        CALLS = _load_calls(LIB_PATH.with_name("_calls.so"), handle)
        _LIB = handle
    return _LIB


def _load_calls(path: Path, handle: ctypes.CDLL):
    """The native host calls of ``path``, bound to the library's entry points; None
    (and, where there is a file, a warning) if they are not for this Python and torch."""
    if not path.exists():
        return None
    want = f"torch {torch.__version__}, Python {sys.version_info[0]}.{sys.version_info[1]}"
    spec = importlib.util.spec_from_file_location(f"{__package__}._calls", path)
    try:
        calls = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(calls)
        built_for = calls.BUILT_FOR
    except (ImportError, AttributeError) as e:
        built_for = str(e)
    if built_for != want:
        warnings.warn(f"{path} is built for something other than {want} ({built_for}): small MXFP4, int8, rotary "
                      f"and per-head norm calls go through Python; build again", RuntimeWarning, stacklevel=2)
        return None
    calls.bind(*(ctypes.cast(getattr(handle, name), _vp).value for name in _CALLS_ENTRIES))
    return calls


class LtxKernelError(RuntimeError):
    """A libltx_hip entry point returned a non-zero status."""

    def __init__(self, name: str, status: int, detail: str = ""):
        msg = lib().ltx_status_string(status).decode()
        super().__init__(f"{name} failed with status {status} ({msg}){': ' + detail if detail else ''}")
        self.status = status


def call(name: str, *args, detail: str = "") -> None:
    status = getattr(lib(), name)(*args)
    if status != 0:
        raise LtxKernelError(name, status, detail)


def launch(device: int, name: str, *args) -> int:
    """Status of an entry point, called with ``device`` current (a launch goes
    to the current device) and that device's current stream as last argument."""
    fn = getattr(_LIB or lib(), name)
    if device == _current_device():
        return fn(*args, _raw_stream(device))
    with torch.cuda.device(device):
        return fn(*args, _raw_stream(device))


def fast_stream(t: torch.Tensor) -> tuple[int, int] | None:
    """(device, its current stream) for a native host call on t's GPU; None
    where t is not on the current GPU."""
    device = t.get_device()
    if device < 0 or device != _current_device():
        return None
    return device, _raw_stream(device)


def launched(result, name: str, detail: str = ""):
    """The result of a native host call that did not pass the call on; a status
    that it came back with raises."""
    if type(result) is int:
        raise LtxKernelError(name, result, detail)
    return result


def same_device(*tensors: torch.Tensor | None) -> int:
    """The GPU index of the given tensors; raises unless all are on one GPU."""
    device = tensors[0].get_device()
    for t in tensors:
        if t is not None and (t.get_device() != device or device < 0):
            raise ValueError(f"expected device tensors on one GPU, got {tensors[0].device} and {t.device}")
    return device


def _axes(t: torch.Tensor) -> list[tuple[int, int]]:
    """(stride in bytes, size) of the axes of more than one entry, outermost last."""
    size = t.element_size()
    return sorted((st * size, n) for st, n in zip(t.stride(), t.shape) if n != 1)


def same_view(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether index for index the two are the same memory."""
    return a.data_ptr() == b.data_ptr() and a.shape == b.shape and all(
        n == 1 or sa == sb for sa, sb, n in zip(a.stride(), b.stride(), a.shape))


def overlaps(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the two may share memory.  Column ranges of one buffer's rows do
    not: with a stride in common, what lies inside it is compared."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    xa, xb = _axes(a), _axes(b)

    def extent(axes, size, below=None):  # bytes from the first element to the end of the last
        return size + sum(st * (n - 1) for st, n in axes if below is None or st < below)

    gap = b.data_ptr() - a.data_ptr()
    if gap >= extent(xa, a.element_size()) or -gap >= extent(xb, b.element_size()):
        return False
    for period in {st for st, _ in xa} & {st for st, _ in xb}:
        if period == 0 or any(st > period and st % period for st, _ in xa + xb):
            continue
        d = gap % period
        if extent(xa, a.element_size(), period) <= d and d + extent(xb, b.element_size(), period) <= period:
            return False
    return True


def self_overlaps(t: torch.Tensor) -> bool:
    """Whether two indices may name the same element."""
    end = t.element_size()
    for st, n in _axes(t) if t.numel() else ():
        if st < end:
            return True
        end += st * (n - 1)
    return False


def ptr(t: torch.Tensor | None) -> int | None:
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError(f"expected a device tensor, got one on {t.device}")
    return t.data_ptr()


def stream_of(t: torch.Tensor) -> int:
    """Handle of the current stream of t's device (the raw handle: building
    torch's Stream object costs the host ~2 us per launch)."""
    if not t.is_cuda:
        raise ValueError(f"expected a device tensor, got one on {t.device}")
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def flat(t: torch.Tensor) -> torch.Tensor:
    """t with its elements in one dense run; t itself where it is dense."""
    return t if t.is_contiguous() else t.reshape(-1).contiguous()


def row_view(t: torch.Tensor, cols: int) -> tuple[torch.Tensor, int]:
    """Return (tensor, row_stride) such that `t` is seen as (rows, cols) rows
    of unit column stride.  Copies only if the layout is not row-uniform."""
    if t.shape[-1] != cols:
        raise ValueError(f"last dim {t.shape[-1]} != {cols}")
    st = t.stride()
    if st[-1] == 1:  # the usual forms: rows of a matrix, or of one batch entry
        if len(st) == 2:
            return t, st[0]
        if len(st) == 3 and t.shape[0] == 1:
            return t, st[1]
    if t.dim() == 1:
        return t.contiguous(), cols
    if t.stride(-1) == 1:
        # leading dims must collapse to one uniform stride
        lead = t.shape[:-1]
        strides = t.stride()[:-1]
        row_stride = strides[-1]
        expect = row_stride
        ok = True
        for size, stride in zip(reversed(lead), reversed(strides)):
            if size != 1 and stride != expect:
                ok = False
                break
            expect = stride * size if size != 1 else expect
        if ok:
            return t, row_stride
    t = t.contiguous()
    return t, cols
