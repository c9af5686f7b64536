"""Workloads of the MXFP4 projections and of rotary positions, as cases that a timing program can
prepare, run and check.

A case is a dict of plain values.  ``prepare(case, seed)`` makes what a program holds before the call (inputs, and
the weights it keeps resident), ``run(state)`` is one pass, ``exact(case, seed)`` the same result in float64,
``work(case)`` the bytes and flops that no implementation can do without.  With ``own`` the pass calls the
package's kernels, without it elementary torch operations in fp32.

Kinds:
  quantize  rows to MXFP4 (blocks of 32, E2M1 codes, E8M0 scales) and their decoded values
  linear    bf16 rows x resident MXFP4 weights (N, K), with a projection's epilogue
  linear_mx MXFP4 rows x MXFP4 weights, the same epilogues
  rotary    rotary positions applied to queries and keys (``transpose``: the gradient's rotation)

MXFP4 data: code bytes (rows, K / 2), the even k in the low nibble, and the E8M0 scales as int32 words
(ceil(K / 128), rows rounded up to 4): word [k // 128, row] holds the four blocks of those 128 k, the first in
its low byte.
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


def listed() -> list[dict]:
    return [
        # the audio stream's rows of a 768x512x65 clip: a launch is a few microseconds
        dict(name="quantize_68x2048", kind="quantize", rows=68, depth=2048, dtype="bf16"),
        # the video rows of a long clip, before a quantised product
        dict(name="quantize_14640x4096", kind="quantize", rows=14640, depth=4096, dtype="bf16"),
        # one row: the weight bytes are everything
        dict(name="linear_1x4096_4096", kind="linear", rows=1, depth=4096, cols=4096, epilogue="bias"),
        # the audio feed-forward's up-projection: few rows, GELU behind it
        dict(name="linear_68x2048_8192_gelu", kind="linear", rows=68, depth=2048, cols=8192, epilogue="gelu"),
        # query, key, value and head-gate columns of a 512x288x65 clip in one product
        dict(name="linear_1296x4096_12320_gates", kind="linear", rows=1296, depth=4096, cols=12320,
             epilogue="gates"),
        # the video feed-forward's down-projection at 768x512x65 with the block's gated residual
        dict(name="linear_3456x16384_4096_residual", kind="linear", rows=3456, depth=16384, cols=4096,
             epilogue="residual"),
        # a prompt's 256 rows, quantised: few tiles
        dict(name="linear_mx_256x4096_8192", kind="linear_mx", rows=256, depth=4096, cols=8192, epilogue="bias"),
        # the up-projection of a 768x512x121 clip with quantised rows: the largest
        dict(name="linear_mx_6144x4096_16384_gelu", kind="linear_mx", rows=6144, depth=4096, cols=16384,
             epilogue="gelu"),
        # one new token far into a sequence, frequencies stretched for a long context
        dict(name="rotary_1_half_yarn", kind="rotary", tokens=1, heads=32, kv_heads=32, head_dim=128, rotary=128,
             layout="half", dtype="bf16", scaling="yarn", start=100003, transpose=False),
        # queries and keys of a 768x512x65 clip's token sequence, neighbouring channels paired
        dict(name="rotary_3456_interleaved", kind="rotary", tokens=3456, heads=32, kv_heads=32, head_dim=128,
             rotary=128, layout="interleaved", dtype="bf16", scaling="none", start=0, transpose=False),
        # the gradient of a half-rotated head, fp32, fewer key heads, an odd length
        dict(name="rotary_14639_partial_grad_fp32", kind="rotary", tokens=14639, heads=32, kv_heads=8, head_dim=64,
             rotary=32, layout="half", dtype="fp32", scaling="linear", start=7, transpose=True),
    ]


def draw(rng) -> dict:
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(("quantize", "linear", "linear", "linear_mx", "linear_mx", "rotary"))
    if kind == "quantize":
        return dict(kind=kind, rows=log_int(1, 14640), depth=32 * log_int(1, 128), dtype=rng.choice(tuple(DTYPES)))
    if kind == "rotary":
        head_dim = rng.choice((64, 128, 80, 96, 256))
        heads = rng.choice((1, 8, 12, 32))
        return dict(kind=kind, tokens=log_int(1, 14640), heads=heads,
                    kv_heads=rng.choice([h for h in (1, 2, 4, 8, 12, 32) if heads % h == 0]), head_dim=head_dim,
                    rotary=rng.choice((head_dim, head_dim // 2, head_dim // 4)),
                    layout=rng.choice(("half", "interleaved")), dtype=rng.choice(tuple(DTYPES)),
                    scaling=rng.choice(("none", "linear", "yarn")), start=log_int(1, 1 << 20),
                    transpose=rng.random() < 0.4)
    while True:
        unit = 64 if kind == "linear" else 128
        case = dict(kind=kind, rows=log_int(1, 6144), depth=unit * log_int(1, 16384 // unit),
                    cols=8 * log_int(4, 2048), epilogue=rng.choice(("bias", "gelu", "gates", "residual")))
        if work(case)["flops"] <= MAX_FLOPS:
            return case


def work(case) -> dict:
    if case["kind"] == "quantize":
        n = case["rows"] * case["depth"]
        size = DTYPES[case["dtype"]].itemsize
        return dict(bytes=n * size + n // 2 + n // 32 + 2 * n, flops=4 * n)
    if case["kind"] == "rotary":
        heads = case["tokens"] * (case["heads"] + case["kv_heads"])
        return dict(bytes=2 * heads * case["head_dim"] * DTYPES[case["dtype"]].itemsize + 4 * case["tokens"],
                    flops=3 * heads * case["rotary"])
    m, k, n = case["rows"], case["depth"], case["cols"]
    rows = m * k * 2 if case["kind"] == "linear" else m * (k // 2 + k // 32)
    extra = m * n * 2 + n * 4 if case["epilogue"] == "residual" else 0
    return dict(bytes=rows + n * (k // 2 + k // 32) + n * 4 + m * n * 2 + extra, flops=2 * m * n * k)


# ---- inputs ---------------------------------------------------------------------------------------------------

def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(rows: int, depth: int, g: torch.Generator) -> torch.Tensor:
    """Normalised rows: unit normal, every 64th channel eight times as large."""
    x = torch.randn(rows, depth, generator=g, device="cuda")
    x[:, ::64] *= 8
    return x


def _block_exponents(blocks: torch.Tensor) -> torch.Tensor:
    """X = floor(log2(max |v|)) - 2 of every block (last axis), clamped to [-127, 127]; -127 for zeros."""
    amax = blocks.abs().amax(-1)
    _, e = torch.frexp(amax)
    return torch.where(amax > 0, (e - 3).clamp(-127, 127), torch.full_like(e, -127))


def _encode(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 rows (R, K) as E2M1 codes (R, K), one per byte, and block exponents (R, K / 32)."""
    rows, depth = x.shape
    blocks = x.view(rows, depth // 32, 32)
    e = _block_exponents(blocks)
    a = torch.ldexp(blocks, -e[..., None]).abs()
    code = ((a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code |= (blocks < 0).byte() << 3
    return code.view(rows, depth), e


def _pack(code: torch.Tensor, e: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Code bytes (R, K / 2) and scale words (ceil(K / 128), R rounded up to 4) int32."""
    rows, blocks = e.shape
    words = (blocks + 3) // 4
    b = torch.zeros(words, (rows + 3) // 4 * 4, 4, dtype=torch.uint8, device=e.device)
    padded = torch.zeros(rows, words * 4, dtype=torch.uint8, device=e.device)
    padded[:, :blocks] = (e + 127).byte()
    b[:, :rows] = padded.view(rows, words, 4).transpose(0, 1)
    return code[:, ::2] | code[:, 1::2] << 4, b.view(torch.int32).squeeze(-1)


def _frequencies(case) -> tuple[torch.Tensor, float]:
    """Angle per position of every pair (fp64) and the factor on cos and sin.  linear: positions divided by 8;
    yarn: slow pairs divided by 16, fast ones kept, a ramp between (betas 32 and 1, original length 4096)."""
    d = case["rotary"]
    inv = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    if case["scaling"] == "linear":
        return (inv / 8).cuda(), 1.0
    if case["scaling"] == "yarn":
        lo, hi = (d * math.log(4096 / (b * 2 * math.pi)) / (2 * math.log(10000.0)) for b in (32, 1))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), d - 1)
        ramp = ((torch.arange(d // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return (inv * (1 - ramp) + inv / 16 * ramp).cuda(), 0.1 * math.log(16) + 1
    return inv.cuda(), 1.0


def prepare(case, seed) -> dict:
    g = _generator(seed)
    if case["kind"] == "quantize":
        return dict(case=case, x=_activations(case["rows"], case["depth"], g).to(DTYPES[case["dtype"]]))
    if case["kind"] == "rotary":
        t, dh, dtype = case["tokens"], case["head_dim"], DTYPES[case["dtype"]]
        q = torch.randn(t, case["heads"], dh, generator=g, device="cuda").to(dtype)
        k = torch.randn(t, case["kv_heads"], dh, generator=g, device="cuda").to(dtype)
        positions = torch.arange(t, dtype=torch.int32, device="cuda") + case["start"]
        inv, factor = _frequencies(case)
        return dict(case=case, q=q, k=k, positions=positions, inv=inv, factor=factor)
    m, k, n = case["rows"], case["depth"], case["cols"]
    s = dict(case=case, bias=torch.randn(n, generator=g, device="cuda") * 0.1)
    w = torch.randn(n, k, generator=g, device="cuda") * k ** -0.5
    s["w"], s["w_scale"] = _pack(*_encode(w))
    x = _activations(m, k, g)
    if case["kind"] == "linear":
        s["x"] = x.bfloat16()
    else:
        s["x"], s["x_scale"] = _pack(*_encode(x))
    if case["epilogue"] == "residual":
        s["residual"] = (2 * torch.randn(m, n, generator=g, device="cuda")).bfloat16()
        s["gate"] = torch.randn(n, generator=g, device="cuda") * 0.5
    return s


# ---- the plain form: fp32, rounded once at the end --------------------------------------------------------------

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _decoded(codes: torch.Tensor, words: torch.Tensor) -> torch.Tensor:
    rows, half = codes.shape
    table = torch.tensor(_E2M1, device=codes.device)
    v = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1).view(rows, half // 16, 32)
    e = words[:, :rows].contiguous().view(torch.uint8).view(-1, rows, 4).transpose(0, 1).reshape(rows, -1)
    return torch.ldexp(v, (e[:, :half // 16].int() - 127)[..., None]).view(rows, half * 2)


def _gate_from(case) -> int:
    """First of the head-gate columns: the last 32 (all of a narrower product's but 8)."""
    return max(case["cols"] - 32, 8)


def _finish(y: torch.Tensor, s: dict) -> torch.Tensor:
    case = s["case"]
    y = y + s["bias"].to(y.dtype)
    if case["epilogue"] == "gelu":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    elif case["epilogue"] == "gates":
        c = _gate_from(case)
        y = torch.cat((y[:, :c], 2 / (1 + torch.exp(-y[:, c:]))), 1)
    elif case["epilogue"] == "residual":
        y = s["residual"].to(y.dtype) + s["gate"].to(y.dtype) * y
    return y


def _rotated(x: torch.Tensor, angle: torch.Tensor, s: dict, work_type: torch.dtype) -> torch.Tensor:
    case = s["case"]
    d = case["rotary"]
    c = (torch.cos(angle) * s["factor"]).to(work_type)[:, None, :]
    n = (torch.sin(angle) * s["factor"]).to(work_type)[:, None, :]
    if case["transpose"]:
        n = -n
    v = x.to(work_type)
    if case["layout"] == "half":
        a, b = v[..., :d // 2], v[..., d // 2:d]
        r = torch.cat((a * c - b * n, b * c + a * n, v[..., d:]), -1)
    else:
        a, b = v[..., 0:d:2], v[..., 1:d:2]
        r = torch.cat((torch.stack((a * c - b * n, b * c + a * n), -1).flatten(-2), v[..., d:]), -1)
    return r


def _plain(s: dict):
    case = s["case"]
    if case["kind"] == "quantize":
        code, e = _encode(s["x"].float())
        _pack(code, e)  # the stored form
        table = torch.tensor(_E2M1, device=code.device)
        v = table[code.int()].view(*e.shape, 32)
        return torch.ldexp(v, e[..., None]).view(code.shape).bfloat16()
    if case["kind"] == "rotary":
        angle = s["positions"].double()[:, None] * s["inv"]
        return tuple(_rotated(s[t], angle, s, torch.float32).to(s[t].dtype) for t in "qk")
    x = s["x"].float() if case["kind"] == "linear" else _decoded(s["x"], s["x_scale"])
    return _finish(x @ _decoded(s["w"], s["w_scale"]).t(), s).bfloat16()


# ---- the package's operators --------------------------------------------------------------------------------------

def _framework(s: dict):
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from ltx_amd.kernels import gemm, rope_ops

    case = s["case"]
    if case["kind"] == "quantize":
        return gemm.dequantize_rows_mxfp4(gemm.quantize_rows_mxfp4(s["x"]))
    if case["kind"] == "rotary":
        return rope_ops.rotary(s["q"], s["k"], s["positions"], s["inv"], layout=case["layout"], factor=s["factor"],
                               transpose=case["transpose"])
    weight = gemm.LinearWeight("mxfp4", s["w"], s["w_scale"], s["bias"])
    x = s["x"] if case["kind"] == "linear" else gemm.Mx4Rows(s["x"], s["x_scale"])
    if case["epilogue"] == "gelu":
        return gemm.linear(x, weight, epilogue=gemm.EPI_GELU)
    if case["epilogue"] == "gates":
        return gemm.linear(x, weight, sigmoid_from=_gate_from(case))
    if case["epilogue"] == "residual":
        return gemm.linear(x, weight, epilogue=gemm.EPI_RESIDUAL, residual=s["residual"], gate=s["gate"])
    return gemm.linear(x, weight)


def run(state):
    return _framework(state) if own else _plain(state)


# ---- float64, from the formats' and the operators' definitions ------------------------------------------------------

def _values64(codes: torch.Tensor, words: torch.Tensor) -> torch.Tensor:
    """E2M1 by its fields: sign, two exponent bits (bias 1, subnormals at 0), one mantissa bit."""
    rows = codes.shape[0]
    nib = torch.empty(rows, codes.shape[1] * 2, dtype=torch.int64, device=codes.device)
    nib[:, 0::2], nib[:, 1::2] = (codes % 16).long(), (codes // 16).long()
    e, m = nib // 2 % 4, (nib % 2).double()
    v = torch.where(e == 0, m / 2, (1 + m / 2) * 2.0 ** (e - 1).double()) * (1 - 2 * (nib // 8)).double()
    w = words[:, :rows].long() % (1 << 32)
    for b in range(0, nib.shape[1], 32):
        scale = (w[b // 128] >> (b // 32 % 4 * 8)) % 256
        v[:, b:b + 32] *= (2.0 ** (scale - 127).double())[:, None]
    return v


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quantize":
        x = s["x"].double().view(case["rows"], -1, 32)
        top = x.abs().amax(-1, keepdim=True)
        step = 2.0 ** (torch.floor(torch.log2(top)) - 2)
        y = x / step
        # E2M1 around |y|: spacing 1/2 below 2, 1 from 2 to 4, 2 above; nearest, ties to even; at most 6
        gap = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0)).double()
        return torch.where(top > 0, (torch.round(y / gap) * gap).clamp(-6, 6) * step,
                           torch.zeros_like(x)).view(case["rows"], -1)
    if case["kind"] == "rotary":
        angle = s["positions"].double()[:, None] * s["inv"]
        turn = torch.polar(torch.full_like(angle, s["factor"]), -angle if case["transpose"] else angle)[:, None]
        out = []
        for t in "qk":
            v, d = s[t].double(), case["rotary"]
            half = case["layout"] == "half"
            z = v[..., :d].unflatten(-1, (2, d // 2)).transpose(-1, -2) if half else v[..., :d].unflatten(-1, (-1, 2))
            z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
            v[..., :d] = (z.transpose(-1, -2) if half else z).flatten(-2)
            out.append(v)
        return tuple(out)
    x = s["x"].double() if case["kind"] == "linear" else _values64(s["x"], s["x_scale"])
    y = torch.addmm(s["bias"].double(), x, _values64(s["w"], s["w_scale"]).t())
    if case["epilogue"] == "gelu":
        y = torch.nn.functional.gelu(y, approximate="tanh")
    elif case["epilogue"] == "gates":
        y[:, _gate_from(case):].sigmoid_().mul_(2)
    elif case["epilogue"] == "residual":
        y = torch.addcmul(s["residual"].double(), s["gate"].double(), y)
    return y
