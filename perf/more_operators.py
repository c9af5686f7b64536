"""Workloads of the int8 projections (8-bit rows times 8-bit weights) and of the per-head norm with rotary
positions, as cases that a timing program can prepare, run and check.

A case is a dict of plain values.  ``prepare(case, seed)`` makes what a program holds before the call (inputs, and
the weights it keeps resident), ``run(state)`` is one pass, ``exact(case, seed)`` the same result in float64,
``work(case)`` the bytes and flops that no implementation can do without.  With ``own`` the pass calls the
package's kernels, without it elementary torch operations in fp32.

Kinds:
  quantize   rows to int8 with a scale per row, and their decoded values
  linear     int8 rows x resident int8 weights (N, K), with a projection's epilogue; the rows come as int8
             (``given`` "int8": several projections of one input share them) or are quantised in the pass
  norm       queries and keys: RMS norm of every head, its weights, rotary positions
  norm_grad  the gradients of both and of the norm weights

int8 data: codes (rows, K) and fp32 scales (rows): scale = max |v| / 127, code = v / scale to the nearest integer,
ties to even, in fp32.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parent.parent / "ltx-2-mlx_amd")
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MAX_FLOPS = 2 * 6144 * 4096 * 16384
EPS = 1e-6


def listed() -> list[dict]:
    return [
        # the audio stream's rows of a 768x512x65 clip: a launch is a few microseconds
        dict(name="quantize_68x2048", kind="quantize", rows=68, depth=2048, dtype="bf16"),
        # the video rows of a long clip, before a quantised product
        dict(name="quantize_14640x4096", kind="quantize", rows=14640, depth=4096, dtype="bf16"),
        # one row: the weight bytes are everything
        dict(name="linear_1x4096_4096", kind="linear", rows=1, depth=4096, cols=4096, epilogue="bias", given="int8"),
        # the audio feed-forward's up-projection: few rows, GELU behind it
        dict(name="linear_68x2048_8192_gelu", kind="linear", rows=68, depth=2048, cols=8192, epilogue="gelu",
             given="int8"),
        # query, key, value and head-gate columns of a 512x288x65 clip in one product, from bf16 rows
        dict(name="linear_1296x4096_12320_gates", kind="linear", rows=1296, depth=4096, cols=12320,
             epilogue="gates", given="bf16"),
        # the video feed-forward's down-projection at 768x512x65 with the block's gated residual
        dict(name="linear_3456x16384_4096_residual", kind="linear", rows=3456, depth=16384, cols=4096,
             epilogue="residual", given="int8"),
        # the up-projection of a 768x512x121 clip: the largest
        dict(name="linear_6144x4096_16384_gelu", kind="linear", rows=6144, depth=4096, cols=16384, epilogue="gelu",
             given="int8"),
        # one new token far into a sequence, fewer key heads, weights held as their difference from one
        dict(name="norm_1_half", kind="norm", tokens=1, heads=32, kv_heads=8, head_dim=128, rotary=128,
             layout="half", dtype="bf16", offset=1.0, weights=True, start=100003),
        # queries and keys of a 768x512x65 clip's token sequence, neighbouring channels paired
        dict(name="norm_3456_interleaved", kind="norm", tokens=3456, heads=32, kv_heads=32, head_dim=128, rotary=128,
             layout="interleaved", dtype="bf16", offset=0.0, weights=True, start=0),
        # a long clip, narrow heads of which half rotates, fp32, an odd length
        dict(name="norm_14639_partial_fp32", kind="norm", tokens=14639, heads=32, kv_heads=8, head_dim=64, rotary=32,
             layout="half", dtype="fp32", offset=0.0, weights=True, start=7),
        # the gradient of a prompt's 257 tokens: few workgroups, a sum over all of them
        dict(name="norm_grad_257_fp32", kind="norm_grad", tokens=257, heads=12, kv_heads=4, head_dim=64, rotary=64,
             layout="half", dtype="fp32", offset=1.0, weights=True, start=0),
        # the gradient at a long clip's length, fewer key heads
        dict(name="norm_grad_14640_half", kind="norm_grad", tokens=14640, heads=32, kv_heads=8, head_dim=128,
             rotary=128, layout="half", dtype="bf16", offset=0.0, weights=True, start=0),
    ]


def draw(rng) -> dict:
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(("quantize", "linear", "linear", "linear", "norm", "norm", "norm_grad", "norm_grad"))
    if kind == "quantize":
        return dict(kind=kind, rows=log_int(1, 14640), depth=16 * log_int(1, 256), dtype=rng.choice(tuple(DTYPES)))
    if kind != "linear":
        head_dim = rng.choice((64, 128, 80, 96, 256))
        heads = rng.choice((1, 8, 12, 32) if head_dim <= 128 else (1, 8, 16))
        return dict(kind=kind, tokens=log_int(1, 14640), heads=heads,
                    kv_heads=rng.choice([h for h in (1, 2, 4, 8, 12, 32) if heads % h == 0]), head_dim=head_dim,
                    rotary=rng.choice((head_dim, head_dim // 2, head_dim // 4)),
                    layout=rng.choice(("half", "interleaved")), dtype=rng.choice(tuple(DTYPES)),
                    offset=rng.choice((0.0, 1.0)), weights=rng.random() < 0.85, start=log_int(1, 1 << 20))
    while True:
        case = dict(kind=kind, rows=log_int(1, 6144), depth=64 * log_int(1, 256), cols=8 * log_int(4, 2048),
                    epilogue=rng.choice(("bias", "gelu", "gates", "residual")), given=rng.choice(("int8", "bf16")))
        if work(case)["flops"] <= MAX_FLOPS:
            return case


def work(case) -> dict:
    if case["kind"] == "quantize":
        n = case["rows"] * case["depth"]
        size = DTYPES[case["dtype"]].itemsize
        return dict(bytes=n * size + n + 4 * case["rows"] + 2 * n, flops=4 * n)
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["depth"], case["cols"]
        rows = m * k + 4 * m if case["given"] == "int8" else 2 * m * k
        extra = m * n * 2 + n * 4 if case["epilogue"] == "residual" else 0
        return dict(bytes=rows + n * k + n * 8 + m * n * 2 + extra, flops=2 * m * n * k)
    channels = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
    moved = 2 if case["kind"] == "norm" else 3
    weights = 8 * case["head_dim"] * (moved - 1) if case["weights"] else 0
    return dict(bytes=moved * channels * DTYPES[case["dtype"]].itemsize + 4 * case["tokens"] + weights,
                flops=(moved * 4 - 2) * channels)


# ---- inputs ---------------------------------------------------------------------------------------------------

def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(rows: int, depth: int, g: torch.Generator) -> torch.Tensor:
    """Normalised rows: unit normal, every 64th channel eight times as large."""
    x = torch.randn(rows, depth, generator=g, device="cuda")
    x[:, ::64] *= 8
    return x


def _to_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 rows as int8 codes and fp32 scales (rows)."""
    scale = x.abs().amax(1) / 127
    q = torch.where(scale[:, None] > 0, torch.round(x / scale[:, None]), torch.zeros_like(x))
    return q.clamp(-127, 127).to(torch.int8), scale


def _inv_freq(rotary: int) -> torch.Tensor:
    return (10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)).cuda()


def prepare(case, seed) -> dict:
    g = _generator(seed)
    if case["kind"] == "quantize":
        return dict(case=case, x=_activations(case["rows"], case["depth"], g).to(DTYPES[case["dtype"]]))
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["depth"], case["cols"]
        s = dict(case=case, bias=torch.randn(n, generator=g, device="cuda") * 0.1)
        s["w"], s["w_scale"] = _to_int8(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5)
        x = _activations(m, k, g).bfloat16()
        if case["given"] == "int8":
            s["x"], s["x_scale"] = _to_int8(x.float())
        else:
            s["x"] = x
        if case["epilogue"] == "residual":
            s["residual"] = (2 * torch.randn(m, n, generator=g, device="cuda")).bfloat16()
            s["gate"] = torch.randn(n, generator=g, device="cuda") * 0.5
        return s
    t, dh, dtype = case["tokens"], case["head_dim"], DTYPES[case["dtype"]]
    s = dict(case=case, positions=torch.arange(t, dtype=torch.int32, device="cuda") + case["start"],
             inv=_inv_freq(case["rotary"]), wq=None, wk=None)
    for name, heads in (("q", case["heads"]), ("k", case["kv_heads"])):
        # a projection's output: heads of different sizes
        size = torch.exp2(torch.randn(heads, 1, generator=g, device="cuda"))
        s[name] = (torch.randn(t, heads, dh, generator=g, device="cuda") * size).to(dtype)
        if case["kind"] == "norm_grad":
            s["g" + name] = (torch.randn(t, heads, dh, generator=g, device="cuda") * 0.1).to(dtype)
        if case["weights"]:
            s["w" + name] = torch.randn(dh, generator=g, device="cuda") * 0.2 + (1.0 - case["offset"])
    return s


# ---- the plain form: fp32, rounded once at the end --------------------------------------------------------------

def _gate_from(case) -> int:
    """First of the head-gate columns: the last 32 (all of a narrower product's but 8)."""
    return max(case["cols"] - 32, 8)


def _finish(y: torch.Tensor, s: dict) -> torch.Tensor:
    case = s["case"]
    y = y + s["bias"]
    if case["epilogue"] == "gelu":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    elif case["epilogue"] == "gates":
        c = _gate_from(case)
        y = torch.cat((y[:, :c], 2 / (1 + torch.exp(-y[:, c:]))), 1)
    elif case["epilogue"] == "residual":
        y = s["residual"].float() + s["gate"] * y
    return y


def _rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, layout: str) -> torch.Tensor:
    d = 2 * cos.shape[-1]
    if layout == "half":
        a, b = x[..., :d // 2], x[..., d // 2:d]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., d:]), -1)
    a, b = x[..., 0:d:2], x[..., 1:d:2]
    return torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2), x[..., d:]), -1)


def _plain(s: dict):
    case = s["case"]
    if case["kind"] == "quantize":
        q, scale = _to_int8(s["x"].float())
        return (q.float() * scale[:, None]).bfloat16(), scale
    if case["kind"] == "linear":
        x, scale = (s["x"], s["x_scale"]) if case["given"] == "int8" else _to_int8(s["x"].float())
        y = x.float() @ s["w"].float().t()
        return _finish(y * scale[:, None] * s["w_scale"], s).bfloat16()
    angle = (s["positions"].double()[:, None] * s["inv"])[:, None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    out, sums = [], []
    for name in "qk":
        x, w = s[name].float(), s["w" + name]
        scale = 1.0 if w is None else w + case["offset"]
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        n = x * r
        if case["kind"] == "norm":
            out.append(_rotate(n * scale, cos, sin, case["layout"]).to(s[name].dtype))
            continue
        gz = _rotate(s["g" + name].float(), cos, -sin, case["layout"])
        gn = gz * scale
        out.append((r * (gn - n * (gn * n).mean(-1, keepdim=True))).to(s[name].dtype))
        sums.append(None if w is None else (gz * n).sum((0, 1), dtype=torch.float64).float())
    return tuple(out + [t for t in sums if t is not None])


# ---- the package's operators --------------------------------------------------------------------------------------

def _framework(s: dict):
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from ltx_amd.kernels import gemm, rope_ops

    case = s["case"]
    if case["kind"] == "quantize":
        rows = gemm.quantize_rows_int8(s["x"])
        return gemm.dequantize_rows_int8(rows), rows.scales
    if case["kind"] == "linear":
        weight = gemm.LinearWeight("int8", s["w"], s["w_scale"], s["bias"])
        x = gemm.Int8Rows(s["x"], s["x_scale"]) if case["given"] == "int8" else gemm.quantize_rows_int8(s["x"])
        if case["epilogue"] == "gelu":
            return gemm.linear(x, weight, epilogue=gemm.EPI_GELU)
        if case["epilogue"] == "gates":
            return gemm.linear(x, weight, sigmoid_from=_gate_from(case))
        if case["epilogue"] == "residual":
            return gemm.linear(x, weight, epilogue=gemm.EPI_RESIDUAL, residual=s["residual"], gate=s["gate"])
        return gemm.linear(x, weight)
    how = dict(eps=EPS, weight_offset=case["offset"], layout=case["layout"])
    if case["kind"] == "norm":
        return rope_ops.headnorm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["positions"], s["inv"], **how)
    grads = rope_ops.headnorm_rotary_grad(s["gq"], s["gk"], s["q"], s["k"], s["wq"], s["wk"], s["positions"],
                                          s["inv"], **how)
    return tuple(t for t in grads if t is not None)


def run(state):
    return _framework(state) if own else _plain(state)


# ---- float64, from the format's and the operators' definitions ------------------------------------------------------

def _codes64(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The int8 format's codes: both of its quotients are fp32 ones (a quotient of fp32 values rounded to fp64 and
    then to fp32 is the fp32 quotient)."""
    scale = (x.abs().max(1, keepdim=True).values / 127.0).float().double()
    q = (x / scale).float().double()
    lower = torch.floor(q)
    up = (q - lower > 0.5) | ((q - lower == 0.5) & (lower % 2 != 0))
    return torch.nan_to_num(lower + up.double()).clamp(-127, 127), scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quantize":
        q, scale = _codes64(s["x"].double())
        return q * scale, scale[:, 0]
    if case["kind"] == "linear":
        q, scale = (s["x"].double(), s["x_scale"].double()[:, None]) if case["given"] == "int8" else _codes64(
            s["x"].double())
        y = torch.addmm(s["bias"].double(), q * scale, (s["w"].double() * s["w_scale"].double()[:, None]).t())
        if case["epilogue"] == "gelu":
            y = torch.nn.functional.gelu(y, approximate="tanh")
        elif case["epilogue"] == "gates":
            y[:, _gate_from(case):].sigmoid_().mul_(2)
        elif case["epilogue"] == "residual":
            y = torch.addcmul(s["residual"].double(), s["gate"].double(), y)
        return y
    turn = torch.exp(1j * (s["positions"].double()[:, None] * s["inv"]))[:, None]
    d, half = case["rotary"], case["layout"] == "half"

    def turned(v):
        z = v[..., :d].unflatten(-1, (2, d // 2)).transpose(-1, -2) if half else v[..., :d].unflatten(-1, (-1, 2))
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
        return torch.cat(((z.transpose(-1, -2) if half else z).flatten(-2), v[..., d:]), -1)

    out, sums = [], []
    for name in "qk":
        leaves = [s[name].double()] + ([] if s["w" + name] is None else [s["w" + name].double()])
        grad = case["kind"] == "norm_grad"
        for t in leaves:
            t.requires_grad_(grad)
        y = leaves[0] / torch.sqrt(leaves[0].square().mean(-1, keepdim=True) + EPS)
        y = turned(y * (leaves[1] + case["offset"]) if len(leaves) > 1 else y)
        if not grad:
            out.append(y)
            continue
        g = torch.autograd.grad(y, leaves, s["g" + name].double())
        out.append(g[0])
        sums.extend(g[1:])
    return tuple(out + sums)
