"""The block-scaled e4m3 operators, as they are measured: the fused residual / RMSNorm / quantiser,
the activation quantisers with one scale per token and 128 columns, and the matrix product that
applies such scales together with one weight scale per 128 x 128 block.

    norm      s = residual + gate * x,  y = s / rms(s) * weight + shift,  codes = e4m3(y / scale)
    quantize  codes = e4m3(f(x) / scale), f the identity, a * g * sigmoid(g) or GELU
    gemm      out[m, n] = sum_b a_scale[m, b] * b_scale[n / 128, b] * sum_{k in block b} a[m, k] b[n, k]
              (+ bias[n]), and residual[m, n] + gate[n] * (.) where the case has a residual

scale = max(absmax * fp32(1/448), 1e-12) over a row, or over each 128 columns of it.  The 8-bit
outputs are returned in their own type, next to their scales.
"""
import math
import sys
from pathlib import Path

import torch

own = False

BLOCK = 128
INV448 = float(torch.tensor(1.0 / 448.0, dtype=torch.float32))
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
MAX_ELEMENTS = 124992 * 4096
MAX_PRODUCT = 124992 * 12288 * 4096
EPS = 1e-6


# ------------------------------------------------------------------------------------- cases
def _norm(M, C, dtype="bf16", blocks=True, residual=True, gate=False, shift=False, samples=1, **name):
    return dict(name, op="norm", M=M, C=C, dtype=dtype, blocks=blocks, residual=residual, gate=gate, shift=shift,
                samples=samples)


def _quantize(M, K, act="none", dtype="bf16", **name):
    return dict(name, op="quantize", M=M, K=K, act=act, dtype=dtype)


def _gemm(M, N, K, out="bf16", bias=False, residual=False, **name):
    return dict(name, op="gemm", M=M, N=N, K=K, out=out, bias=bias, residual=residual)


def listed():
    return [
        # one conditioning token through a block's second norm: latency
        _norm(1, 4096, name="norm 1 x 4096"),
        # a short text prompt at the width of the fp8 model tests, fp32 stream, one scale per token
        _norm(259, 5376, dtype="fp32", blocks=False, name="norm 259 x 5376 fp32"),
        # a whole video's tokens: gated residual, adaLN modulation of two samples, block scales
        _norm(124992, 4096, gate=True, shift=True, samples=2, name="norm 124992 x 4096"),
        # one token's attention output before the output projection
        _quantize(1, 4096, name="quantize 1 x 4096"),
        # a prompt's SwiGLU before the down projection
        _quantize(259, 14336, act="swiglu", name="swiglu 259 x 14336"),
        # a quarter of a video's tokens through the DiT feed-forward's GELU
        _quantize(31248, 16384, act="gelu", name="gelu 31248 x 16384"),
        # one token through a square projection: the weight's bytes and latency
        _gemm(1, 4096, 4096, name="gemm 1 x 4096 x 4096"),
        # a few tokens (prompt heads, timestep embeddings of a batch) through an up projection
        _gemm(24, 14336, 5376, bias=True, name="gemm 24 x 14336 x 5376"),
        # a prompt through the fused SwiGLU projection of the fp8 model tests
        _gemm(259, 28672, 5376, name="gemm 259 x 28672 x 5376"),
        # ragged on every side, fp32 out
        _gemm(1000, 392, 4112, out="fp32", bias=True, name="gemm 1000 x 392 x 4112"),
        # a latent frame group through the down projection with its gated residual
        _gemm(5208, 4096, 16384, residual=True, name="gemm 5208 x 4096 x 16384"),
        # a whole video's tokens through the fused q, k, v projection
        _gemm(124992, 12288, 4096, name="gemm 124992 x 12288 x 4096"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "gemm", "gemm"])
    if op == "norm":
        C = _log(rng, 100, 16384)
        M = _log(rng, 1, min(124992, MAX_ELEMENTS // C))
        samples = rng.choice([1, 1, 2, 3])
        M = max(samples, M // samples * samples)
        residual = rng.random() < 0.7
        return _norm(M, C, dtype=rng.choice(["bf16", "bf16", "fp32"]), blocks=rng.random() < 0.7, residual=residual,
                     gate=residual and rng.random() < 0.5, shift=rng.random() < 0.5, samples=samples)
    if op == "quantize":
        K = _log(rng, 100, 16384)
        M = _log(rng, 1, min(124992, MAX_ELEMENTS // K))
        return _quantize(M, K, act=rng.choice(["none", "swiglu", "gelu"]), dtype=rng.choice(["bf16", "bf16", "fp32"]))
    N, K = _log(rng, 64, 28672), 16 * _log(rng, 4, 1024)
    M = _log(rng, 1, min(124992, MAX_PRODUCT // (N * K)))
    return _gemm(M, N, K, out=rng.choice(["bf16", "bf16", "fp32"]), bias=rng.random() < 0.5,
                 residual=rng.random() < 0.3)


# ------------------------------------------------------------------------------------ inputs
def _blocks(n):
    return -(-n // BLOCK)


def _absmax(y, blocks):
    """absmax of each row [M, 1], or of each 128 columns of it [M, ceil(K / 128)]."""
    if not blocks:
        return y.abs().amax(dim=1, keepdim=True)
    M, K = y.shape
    y = torch.nn.functional.pad(y, (0, _blocks(K) * BLOCK - K))
    return y.view(M, -1, BLOCK).abs().amax(dim=2)


def _spread(scale, K):
    """Scales [M, blocks] as columns [M, K]."""
    return scale.repeat_interleave(BLOCK, dim=1)[:, :K] if scale.shape[1] > 1 else scale


def _quantized(y, blocks):
    scale = (_absmax(y, blocks) * INV448).clamp_min(1e-12)
    return (y / _spread(scale, y.shape[1])).to(torch.float8_e4m3fn), scale


def _activations(M, K, g):
    """Hidden states: N(0, 1) with a log-normal magnitude per token."""
    size = torch.empty(M, 1, device="cuda").log_normal_(0.0, 0.5, generator=g)
    return torch.randn(M, K, device="cuda", generator=g).mul_(size)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=c)
    if c["op"] == "norm":
        dt = DTYPES[c["dtype"]]
        s["x"] = _activations(c["M"], c["C"], g).to(dt)
        s["residual"] = _activations(c["M"], c["C"], g).to(dt) if c["residual"] else None
        rows = (c["samples"], c["C"]) if c["samples"] > 1 else (c["C"],)
        s["weight"] = 1 + 0.1 * torch.randn(rows, device="cuda", generator=g)
        s["gate"] = 0.5 * torch.randn(rows, device="cuda", generator=g) if c["gate"] else None
        s["shift"] = 0.1 * torch.randn(rows, device="cuda", generator=g) if c["shift"] else None
    elif c["op"] == "quantize":
        s["x"] = _activations(c["M"], 2 * c["K"] if c["act"] == "swiglu" else c["K"], g).to(DTYPES[c["dtype"]])
    else:
        M, N, K = c["M"], c["N"], c["K"]
        s["a"], s["a_scale"] = _quantized(_activations(M, K, g), True)
        w = 0.02 * torch.randn(N, K, device="cuda", generator=g)
        # one scale per 128 x 128 block of the weight
        rows = torch.nn.functional.pad(_absmax(w, True), (0, 0, 0, _blocks(N) * BLOCK - N))
        s["b_scale"] = (rows.view(-1, BLOCK, _blocks(K)).amax(dim=1) * INV448).clamp_min(1e-12)
        s["b"] = (w / _spread(s["b_scale"].repeat_interleave(BLOCK, dim=0)[:N], K)).to(torch.float8_e4m3fn)
        s["bias"] = torch.randn(N, device="cuda", generator=g) if c["bias"] else None
        s["residual"] = _activations(M, N, g).to(DTYPES[c["out"]]) if c["residual"] else None
        s["gate"] = 0.5 * torch.randn(N, device="cuda", generator=g) if c["residual"] else None
    return s


# --------------------------------------------------------------------------------- plain form
def _rows(v, M):
    """A vector [C] or one per sample [S, C] as rows that broadcast over [M, C]."""
    return v if v is None or v.dim() == 1 else v.repeat_interleave(M // v.shape[0], dim=0)


def _plain(s):
    c = s["case"]
    if c["op"] == "norm":
        M, y, summed = c["M"], s["x"].float(), None
        if s["residual"] is not None:
            y = s["residual"].float() + (y if s["gate"] is None else _rows(s["gate"], M) * y)
            summed = y.to(s["x"].dtype)
        y = y * torch.rsqrt(y.square().mean(dim=1, keepdim=True) + EPS) * _rows(s["weight"], M)
        if s["shift"] is not None:
            y = y + _rows(s["shift"], M)
        codes, scale = _quantized(y, c["blocks"])
        return codes, scale, summed
    if c["op"] == "quantize":
        y = s["x"].float()
        if c["act"] == "swiglu":
            a, gate = y.chunk(2, dim=1)
            y = a * gate / (1 + torch.exp(-gate))
        elif c["act"] == "gelu":
            y = 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5))
        return _quantized(y, True)
    N, K = c["N"], c["K"]
    a = s["a"].float() * _spread(s["a_scale"], K)
    b = s["b"].float() * _spread(s["b_scale"].repeat_interleave(BLOCK, dim=0)[:N], K)
    out = a @ b.T
    if s["bias"] is not None:
        out = out + s["bias"]
    if s["residual"] is not None:
        out = s["residual"].float() + s["gate"] * out
    return out.to(DTYPES[c["out"]])


# ------------------------------------------------------------------------- the framework's calls
def _fp8_linear():
    root = str(Path(__file__).resolve().parents[1] / "spark-h3_b200")
    if root not in sys.path:
        sys.path.insert(1, root)
    from spark_h3_b200 import fp8_linear

    return fp8_linear


def _own(s):
    c, ops = s["case"], sys.modules.get("spark_h3_b200.fp8_linear") or _fp8_linear()
    if c["op"] == "norm":
        return ops.add_rms_norm_quantize(s["x"], s["weight"], s["residual"], gate=s["gate"], shift=s["shift"], eps=EPS,
                                         blocks=c["blocks"])
    if c["op"] == "quantize":
        if c["act"] == "swiglu":
            return ops.swiglu_quantize_blocks(s["x"])
        if c["act"] == "gelu":
            return ops.gelu_quantize_blocks(s["x"])
        return ops.quantize_blocks(s["x"])
    return ops.fp8_gemm_blocks(s["a"], s["a_scale"], s["b"], s["b_scale"], s["bias"], residual=s["residual"],
                               gate=s["gate"], out_dtype=DTYPES[c["out"]])


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# --------------------------------------------------------------------------------- work, exact
def work(case):
    c = case
    if c["op"] == "gemm":
        M, N, K = c["M"], c["N"], c["K"]
        size = DTYPES[c["out"]].itemsize
        nbytes = M * K + N * K + 4 * (M + _blocks(N)) * _blocks(K) + M * N * size
        nbytes += 4 * N * (c["bias"] + c["residual"]) + M * N * size * c["residual"]
        return {"bytes": nbytes, "flops": 2 * M * N * K}
    M, size = c["M"], DTYPES[c["dtype"]].itemsize
    if c["op"] == "quantize":
        K, reads = c["K"], 2 if c["act"] == "swiglu" else 1
        return {"bytes": M * K * (reads * size + 1) + 4 * M * _blocks(K),
                "flops": M * K * {"none": 2, "swiglu": 7, "gelu": 6}[c["act"]]}
    C = c["C"]
    nbytes = M * C * ((3 if c["residual"] else 1) * size + 1) + 4 * M * (_blocks(C) if c["blocks"] else 1)
    nbytes += 4 * C * c["samples"] * (1 + c["gate"] + c["shift"])
    return {"bytes": nbytes, "flops": M * C * (7 + 2 * c["residual"])}


def exact(case, seed):
    """The same in 64 bits.  In the place of the 8-bit codes stands the quotient that they round."""
    c, s = case, prepare(case, seed)
    if c["op"] == "gemm":
        M, N, K = c["M"], c["N"], c["K"]
        acc = torch.zeros(M, N, dtype=torch.float64, device="cuda")
        for kb in range(_blocks(K)):
            k = slice(kb * BLOCK, min(K, (kb + 1) * BLOCK))
            part = s["a"][:, k].double() @ s["b"][:, k].double().T
            part *= s["a_scale"][:, kb, None].double()
            for nb in range(_blocks(N)):
                n = slice(nb * BLOCK, min(N, (nb + 1) * BLOCK))
                acc[:, n].add_(part[:, n] * s["b_scale"][nb, kb].double())
        if s["bias"] is not None:
            acc += s["bias"].double()
        if s["residual"] is not None:
            acc = s["residual"].double() + s["gate"].double() * acc
        return acc
    y, summed = s["x"].double(), None
    if c["op"] == "norm":
        per = c["M"] // c["samples"]
        vec = {k: None if s[k] is None else s[k].double().view(c["samples"], 1, c["C"])
               for k in ("weight", "gate", "shift")}
        y = y.view(c["samples"], per, c["C"])
        if s["residual"] is not None:
            if vec["gate"] is not None:
                y = y * vec["gate"]
            y = y + s["residual"].double().view_as(y)
            summed = y.reshape(c["M"], c["C"]).clone()
        y = y / torch.sqrt(torch.linalg.vector_norm(y, dim=2, keepdim=True) ** 2 / c["C"] + EPS)
        y = y * vec["weight"]
        if vec["shift"] is not None:
            y = y + vec["shift"]
        y = y.reshape(c["M"], c["C"])
    elif c["act"] == "swiglu":
        y = y[:, :c["K"]] * y[:, c["K"]:] * torch.sigmoid(y[:, c["K"]:])
    elif c["act"] == "gelu":
        y = y * torch.special.ndtr(y)
    width = BLOCK if c.get("blocks", True) else y.shape[1]
    scale = torch.stack([part.abs().amax(dim=1) for part in y.split(width, dim=1)], dim=1) / 448.0
    scale = scale.clamp_min(1e-12)
    codes = torch.cat([part / scale[:, i, None] for i, part in enumerate(y.split(width, dim=1))], dim=1)
    return (codes, scale, summed) if c["op"] == "norm" else (codes, scale)
