"""QK-RMSNorm + split RoPE (in place), the RoPE table layout, rotary
positions without a norm (:func:`rotary`) and after a norm of every head
(:func:`headnorm_rotary`, :func:`headnorm_rotary_grad`).

Replaces the ``q_norm``/``k_norm`` + ``apply_rotary_emb`` sequence of
``Attention.__call__`` (model/transformer/attention.py:578-584) with one HIP
launch per attention call.  The kernel reads the cos/sin tables token-major,
(T, D/2) fp32: the reference's (1, H, T, dh/2) tables transposed once when
they are built (rope.py:274-283).
"""

from __future__ import annotations

import math
import struct

import torch

from .. import _lib


def qknorm_rope_(q: torch.Tensor, wq: torch.Tensor, pe_q: tuple | None,
                 k: torch.Tensor, wk: torch.Tensor, pe_k: tuple | None,
                 heads: int, eps: float = 1e-6) -> None:
    """In-place ``q = rope(q_norm(q), pe_q)``, ``k = rope(k_norm(k), pe_k)``.

    q: (Tq, D) bf16 rows (any row stride, unit column stride); k: (Tk, D).
    wq/wk: fp32 (D).  pe_*: (cos, sin) fp32 (T, D/2), the factored form
    (cos_f, sin_f, idx) of ``rope.factor_tables_np`` -- stacked per-axis rows
    (R, D/2) and int32 (T, axes) row indices -- or None for no RoPE.
    """
    d = q.shape[-1]
    if k.shape[-1] != d:
        raise ValueError(f"q/k inner dims differ: {d} vs {k.shape[-1]}")
    head_dim = d // heads
    qv, qs = _lib.row_view(q, d)
    kv, ks = _lib.row_view(k, d)
    if qv.data_ptr() != q.data_ptr() or kv.data_ptr() != k.data_ptr():
        raise ValueError("qknorm_rope_ works in place: q/k must be row-strided views")
    tq = q.numel() // d if q.dim() > 1 else 1
    tk = k.numel() // d if k.dim() > 1 else 1
    def table(name, pe, rows):
        if pe is None:
            return None, None, None, 1, 0
        cos, sin = pe[0], pe[1]
        if cos.dtype != torch.float32 or cos.shape[-1] != d // 2 or sin.shape != cos.shape:
            raise ValueError(f"{name} tables must be fp32 (R, {d // 2}), got {tuple(cos.shape)}")
        tab_rows = cos.numel() // (d // 2)
        if len(pe) == 2:
            if tab_rows < rows:
                raise ValueError(f"{name} table covers {tab_rows} of {rows} rows")
            return cos, sin, None, 1, tab_rows
        idx = pe[2]
        if idx.dtype != torch.int32 or idx.dim() != 2 or idx.shape[0] < rows or not 1 <= idx.shape[1] <= 3:
            raise ValueError(f"{name} row index must be int32 (T, axes <= 3) covering {rows} rows")
        return cos, sin, idx.contiguous(), idx.shape[1], tab_rows

    cq, sq, iq, aq, rq = table("pe_q", pe_q, tq)
    ck, sk, ik, ak, rk = table("pe_k", pe_k, tk)
    if iq is None and ik is None:
        _lib.call(
            "ltx_qknorm_rope_bf16",
            _lib.ptr(qv), qs, tq, _lib.ptr(wq), _lib.ptr(cq), _lib.ptr(sq),
            _lib.ptr(kv), ks, tk, _lib.ptr(wk), _lib.ptr(ck), _lib.ptr(sk),
            d, head_dim, float(eps), _lib.stream_of(q),
            detail=f"Tq={tq} Tk={tk} D={d} heads={heads}",
        )
        return
    _lib.call(
        "ltx_qknorm_rope_axes_bf16",
        _lib.ptr(qv), qs, tq, _lib.ptr(wq), _lib.ptr(cq), _lib.ptr(sq), _lib.ptr(iq), aq, rq,
        _lib.ptr(kv), ks, tk, _lib.ptr(wk), _lib.ptr(ck), _lib.ptr(sk), _lib.ptr(ik), ak, rk,
        d, head_dim, float(eps), _lib.stream_of(q),
        detail=f"Tq={tq} Tk={tk} D={d} heads={heads} axes={aq}/{ak}",
    )


def tables_from_reference_layout(cos: torch.Tensor, sin: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(B=1, H, T, dh/2) reference tables -> token-major (T, H*dh/2) fp32."""
    if cos.dim() != 4 or cos.shape[0] != 1:
        raise ValueError(f"expected (1, H, T, dh/2) tables, got {tuple(cos.shape)}")
    _, h, t, half = cos.shape
    def tm(a):
        return a[0].permute(1, 0, 2).reshape(t, h * half).float().contiguous()
    return tm(cos), tm(sin)


ROTARY_LAYOUTS = ("half", "interleaved")
ROTARY_SCALINGS = ("none", "linear", "ntk", "yarn")
_ROTARY_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_POSITION_DTYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2, torch.float64: 3}


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, *, scaling: str = "none", stretch: float = 1.0,
                       original_length: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0,
                       device="cuda") -> tuple[torch.Tensor, float]:
    """What :func:`rotary` takes as ``inv_freq`` and ``factor``: the angle per
    position of every channel pair, theta^(-2i/rotary_dim), fp64 on ``device``,
    and the factor on the rotated values.

    ``scaling`` adapts them to sequences ``stretch`` times ``original_length``:
    "linear" divides every frequency by it; "ntk" raises theta so that the
    slowest one is; "yarn" divides the pairs with fewer than ``beta_slow``
    turns over the original length, keeps those with more than ``beta_fast``,
    blends linearly between, and gives the factor 0.1 ln(stretch) + 1.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if scaling not in ROTARY_SCALINGS:
        raise ValueError(f"scaling must be one of {ROTARY_SCALINGS}, got {scaling!r}")
    if not (theta > 1.0 and stretch >= 1.0 and original_length > 0):
        raise ValueError(f"theta > 1, stretch >= 1 and original_length > 0 wanted, got {theta}, {stretch}, "
                         f"{original_length}")
    d = rotary_dim
    if scaling == "ntk" and d > 2:
        theta = theta * stretch ** (d / (d - 2))
    inv = theta ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    factor = 1.0
    if scaling == "linear":
        inv = inv / stretch
    elif scaling == "yarn" and stretch > 1.0:
        def pair(turns: float) -> float:  # the (fractional) pair with this many turns over the original length
            return d * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(theta))

        lo, hi = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), d - 1)
        ramp = ((torch.arange(d // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        inv = inv * (1 - ramp) + inv / stretch * ramp
        factor = 0.1 * math.log(stretch) + 1.0
    return inv.to(device), factor


_ROTARY_ROWS = struct.Struct("9q").pack  # ltx_rotary_rows: x, its strides, out, its strides, heads


def _rotary_side(name: str, x: torch.Tensor, out: torch.Tensor | None) -> tuple[bytes, torch.Tensor]:
    shape, st = x.shape, x.stride()
    if out is None:
        out = x.new_empty(shape)  # dense, whatever the strides of x
    elif out.shape != shape or out.dtype is not x.dtype:
        raise ValueError(f"{name}'s out must be {x.dtype} {tuple(shape)}, got {out.dtype} {tuple(out.shape)}")
    elif _lib.self_overlaps(out):
        raise ValueError(f"{name}'s out has one element in several places")
    so = out.stride()
    if (st[-1] != 1 or so[-1] != 1) and shape[-1] > 1:
        raise ValueError(f"{name} and its out must have unit channel stride")
    if len(st) == 3:
        rows = _ROTARY_ROWS(x.data_ptr(), 0, st[0], st[1], out.data_ptr(), 0, so[0], so[1], shape[1])
    else:
        rows = _ROTARY_ROWS(x.data_ptr(), st[0], st[1], st[2], out.data_ptr(), so[0], so[1], so[2], shape[2])
    return rows, out


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *,
           layout: str = "half", factor: float = 1.0, transpose: bool = False,
           out: tuple[torch.Tensor, torch.Tensor | None] | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Rotary positions of queries and keys, one launch: returns (q', k').

    q: (T, H, dh) or (B, T, H, dh) bf16, fp16 or fp32, any strides but the
    channels'; k likewise with its own number of heads, or None.  The first
    2 * len(inv_freq) channels of a head rotate, the others are copied:
    channels (i, i + d/2) in the "half" layout, (2i, 2i+1) "interleaved" -- the
    reference's split and interleaved forms (model/transformer/rope.py:16-89)
    -- by the angle positions * inv_freq[i], the same for all heads, scaled by ``factor``
    (:func:`rotary_frequencies`).  positions: (T) for every sequence of the
    batch, or (B, T); int32, int64, fp32 or fp64.  ``transpose`` rotates back
    (times ``factor`` again): with the outputs' gradients for q and k it gives
    the inputs' gradients.  ``out`` may be (q, k) itself (in place);
    its tensors must not overlap the others in any other way.
    """
    if layout not in ROTARY_LAYOUTS:
        raise ValueError(f"layout must be one of {ROTARY_LAYOUTS}, got {layout!r}")
    flags = (_lib.ROTARY_INTERLEAVED if layout == "interleaved" else 0) | (_lib.ROTARY_TRANSPOSE if transpose else 0)
    oq, ok = out if out is not None else (None, None)
    if _lib.CALLS is not None:
        where = _lib.fast_stream(q)
        rotated = None if where is None else _lib.CALLS.rotary(q, k, positions, inv_freq, flags, factor, oq, ok, *where)
        if rotated is not None:
            return _lib.launched(rotated, "ltx_rotary")
    shape = q.shape
    dtype = _ROTARY_DTYPES.get(q.dtype)
    if dtype is None or not 3 <= len(shape) <= 4:
        raise ValueError(f"q must be (T, H, dh) or (B, T, H, dh) in bf16, fp16 or fp32, got {q.dtype} "
                         f"{tuple(shape)}")
    *lead, _, dh = shape
    if k is not None:
        *lead_k, _, dk = k.shape
        if k.dtype is not q.dtype or lead_k != lead or dk != dh:
            raise ValueError(f"k {k.dtype} {tuple(k.shape)} does not go with q {q.dtype} {tuple(shape)}")
    batch, tokens = lead if len(lead) == 2 else (1, lead[0])
    if inv_freq.dtype is not torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous fp64 vector (rotary_frequencies)")
    d = 2 * inv_freq.numel()
    if not 2 <= d <= dh:
        raise ValueError(f"{d} rotary channels do not fit heads of {dh}")
    pos_type, pos_shape = _POSITION_DTYPES.get(positions.dtype), positions.shape
    if pos_type is None or (pos_shape != (tokens,) and pos_shape != (batch, tokens)):
        raise ValueError(f"positions must be int32, int64, fp32 or fp64 ({tokens},) or ({batch}, {tokens}), got "
                         f"{positions.dtype} {tuple(pos_shape)}")
    if not positions.is_contiguous():
        positions = positions.contiguous()
    if k is None and ok is not None:
        raise ValueError("out has a tensor for k, but there is no k")
    sq, oq = _rotary_side("q", q, oq)
    sk, ok = _rotary_side("k", k, ok) if k is not None else (None, None)
    if out is not None:
        # workgroups read and write in any order: an output may be its own input, and
        # must keep off everything else that is read or written
        for mine, x, other, y in ((oq, q, ok, k), (ok, k, oq, q)):
            if mine is not None and (
                    (not _lib.same_view(mine, x) and _lib.overlaps(mine, x)) or
                    any(t is not None and _lib.overlaps(mine, t) for t in (other, y, positions, inv_freq))):
                raise ValueError("an output of rotary overlaps another tensor of the call")
    device = _lib.same_device(q, k, positions, inv_freq, oq, ok)
    if batch * tokens == 0:
        return oq, ok
    st = _lib.launch(device, "ltx_rotary", sq, sk, dtype, batch, tokens, dh, d, positions.data_ptr(), pos_type,
                     tokens if len(pos_shape) == 2 else 0, inv_freq.data_ptr(), factor, flags)
    if st:
        raise _lib.LtxKernelError("ltx_rotary", st, f"{q.dtype} B={batch} T={tokens} dh={dh} rotary={d}")
    return oq, ok


_HEADNORM_ROWS = struct.Struct("15q").pack  # ltx_headnorm_rows: x, out, g with their strides, weight, dweight, heads


def _head_strides(name: str, t: torch.Tensor) -> tuple[int, int, int]:
    """Strides of batch, token and head."""
    st = t.stride()
    if st[-1] != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must have unit channel stride")
    return (0, st[0], st[1]) if len(st) == 3 else (st[0], st[1], st[2])


def _headnorm(name: str, q, k, gq, gk, wq, wk, positions, inv_freq, eps, weight_offset, layout, factor, out):
    """Both calls of the per-head norm (gradients: gq is given): checks, outputs, launch."""
    if layout not in ROTARY_LAYOUTS:
        raise ValueError(f"layout must be one of {ROTARY_LAYOUTS}, got {layout!r}")
    grad = gq is not None
    flags = _lib.ROTARY_INTERLEAVED if layout == "interleaved" else 0
    given = out if out is not None else (None, None)
    if _lib.CALLS is not None and positions is not None:
        where = _lib.fast_stream(q)
        if where is not None:
            args = (q, k, wq, wk, positions, inv_freq, flags, factor, eps, weight_offset, *given, *where)
            done = _lib.CALLS.headnorm_grad(gq, gk, *args) if grad else _lib.CALLS.headnorm(*args)
            if done is not None:
                return _lib.launched(done, name)
    shape = q.shape
    dtype = _ROTARY_DTYPES.get(q.dtype)
    if dtype is None or not 3 <= len(shape) <= 4:
        raise ValueError(f"q must be (T, H, dh) or (B, T, H, dh) in bf16, fp16 or fp32, got {q.dtype} {tuple(shape)}")
    *lead, _, dh = shape
    if k is None:
        if wk is not None or gk is not None:
            raise ValueError("weights or a gradient for k, but there is no k")
    else:
        *lead_k, _, dk = k.shape
        if k.dtype is not q.dtype or lead_k != lead or dk != dh:
            raise ValueError(f"k {k.dtype} {tuple(k.shape)} does not go with q {q.dtype} {tuple(shape)}")
    batch, tokens = lead if len(lead) == 2 else (1, lead[0])
    if (positions is None) != (inv_freq is None):
        raise ValueError("positions and inv_freq go together")
    d, pos_type, pos_batch = 0, 0, 0
    if positions is not None:
        if inv_freq.dtype is not torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
            raise ValueError("inv_freq must be a contiguous fp64 vector (rotary_frequencies)")
        d = 2 * inv_freq.numel()
        if not 2 <= d <= dh:
            raise ValueError(f"{d} rotary channels do not fit heads of {dh}")
        pos_type, pos_shape = _POSITION_DTYPES.get(positions.dtype), positions.shape
        if pos_type is None or (pos_shape != (tokens,) and pos_shape != (batch, tokens)):
            raise ValueError(f"positions must be int32, int64, fp32 or fp64 ({tokens},) or ({batch}, {tokens}), got "
                             f"{positions.dtype} {tuple(pos_shape)}")
        if not positions.is_contiguous():
            positions = positions.contiguous()
        pos_batch = tokens if len(pos_shape) == 2 else 0
    elif factor != 1.0:
        raise ValueError("a factor belongs to the rotation, which has no positions")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if k is None and given[1] is not None:
        raise ValueError("out has a tensor for k, but there is no k")
    sides = []
    for n, x, g, w, o in (("q", q, gq, wq, given[0]), ("k", k, gk, wk, given[1])):
        if x is None:
            sides.append((None, None, None, None, None))
            continue
        if w is not None and (w.dtype is not torch.float32 or w.shape != (dh,) or not w.is_contiguous()):
            raise ValueError(f"the norm weights of {n} must be {dh} contiguous fp32 values")
        if grad and (g is None or g.dtype is not x.dtype or g.shape != x.shape):
            raise ValueError(f"the gradient of {n}' must be {x.dtype} {tuple(x.shape)}, got "
                             f"{None if g is None else (g.dtype, tuple(g.shape))}")
        if o is None:
            o = x.new_empty(x.shape)  # dense, whatever the strides of x
        elif o.shape != x.shape or o.dtype is not x.dtype:
            raise ValueError(f"{n}'s out must be {x.dtype} {tuple(x.shape)}, got {o.dtype} {tuple(o.shape)}")
        elif _lib.self_overlaps(o):
            raise ValueError(f"{n}'s out has one element in several places")
        dw = x.new_empty(dh, dtype=torch.float32) if grad and w is not None else None
        rows = _HEADNORM_ROWS(x.data_ptr(), *_head_strides(n, x), o.data_ptr(), *_head_strides(f"{n}'s out", o),
                              g.data_ptr() if grad else 0, *(_head_strides(f"the gradient of {n}'", g) if grad else (0, 0, 0)),
                              0 if w is None else w.data_ptr(), 0 if dw is None else dw.data_ptr(), x.shape[-2])
        sides.append((rows, o, dw, x, g))
    (rq, oq, dwq, _, _), (rk, ok, dwk, _, _) = sides
    if out is not None:
        # workgroups read and write in any order: an output may be its own input (or its
        # gradient), and must keep off everything else that is read or written
        for i, (mine, own) in enumerate(((given[0], (q, gq)), (given[1], (k, gk)))):
            if mine is None:
                continue
            others = [t for t in (*(sides[1 - i][3:]), sides[1 - i][1], wq, wk, positions, inv_freq) if t is not None]
            if any(t is not None and not _lib.same_view(mine, t) and _lib.overlaps(mine, t) for t in own) or any(
                    _lib.overlaps(mine, t) for t in others):
                raise ValueError("an output of the per-head norm overlaps another tensor of the call")
    device = _lib.same_device(q, k, gq, gk, wq, wk, positions, inv_freq, oq, ok)
    args = [rq, rk, dtype, batch, tokens, dh, d, None if positions is None else positions.data_ptr(), pos_type, pos_batch,
            None if inv_freq is None else inv_freq.data_ptr(), factor, eps, weight_offset, flags]
    if grad:
        sums = dwq is not None or dwk is not None
        if batch * tokens == 0 and not sums:
            return oq, ok, dwq, dwk
        size = _lib.lib().ltx_headnorm_rotary_grad_workspace_bytes(dh) if sums else 0
        work = q.new_empty(size, dtype=torch.uint8) if sums else None
        args += [None if work is None else work.data_ptr(), size]
    elif batch * tokens == 0:
        return oq, ok
    st = _lib.launch(device, name, *args)
    if st:
        raise _lib.LtxKernelError(name, st, f"{q.dtype} B={batch} T={tokens} dh={dh} rotary={d}")
    return (oq, ok, dwq, dwk) if grad else (oq, ok)


def headnorm_rotary(q: torch.Tensor, k: torch.Tensor | None, wq: torch.Tensor | None, wk: torch.Tensor | None,
                    positions: torch.Tensor | None, inv_freq: torch.Tensor | None, *, eps: float = 1e-6,
                    weight_offset: float = 0.0, layout: str = "half", factor: float = 1.0,
                    out: tuple[torch.Tensor, torch.Tensor | None] | None = None
                    ) -> tuple[torch.Tensor, torch.Tensor | None]:
    """RMS norm of every query and key head and its rotary position, one launch:
    returns (q', k') = rotary(r x (weight_offset + w)), r = (mean over the head of
    x^2 + eps)^-1/2, all in fp32 and rounded once.

    q, k, positions, inv_freq, layout and factor as in :func:`rotary`;
    positions and inv_freq None: the norm alone.  wq / wk: fp32 (dh), the same for
    all heads (``weight_offset`` 1 for weights held as their difference from one),
    or None for r x alone.  ``out`` may be (q, k) itself (in place); its tensors
    must not overlap the others in any other way.
    """
    return _headnorm("ltx_headnorm_rotary", q, k, None, None, wq, wk, positions, inv_freq, eps, weight_offset, layout,
                     factor, out)


def headnorm_rotary_grad(gq: torch.Tensor, gk: torch.Tensor | None, q: torch.Tensor, k: torch.Tensor | None,
                         wq: torch.Tensor | None, wk: torch.Tensor | None, positions: torch.Tensor | None,
                         inv_freq: torch.Tensor | None, *, eps: float = 1e-6, weight_offset: float = 0.0,
                         layout: str = "half", factor: float = 1.0,
                         out: tuple[torch.Tensor, torch.Tensor | None] | None = None
                         ) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """The gradients of :func:`headnorm_rotary`: from those of its results, gq and
    gk, and its inputs returns (dq, dk, dwq, dwk), the norm weights' in fp32
    (None where there are none), summed over batch, tokens and heads in a fixed
    order.  ``out``: where dq and dk go; each may be its own gradient or input (q and k
    are read, so an output over them ends their use)."""
    if gq is None:
        raise ValueError("headnorm_rotary_grad needs the gradient of q'")
    return _headnorm("ltx_headnorm_rotary_grad", q, k, gq, gk, wq, wk, positions, inv_freq, eps, weight_offset, layout,
                     factor, out)
