"""e4m3 linears on the B200 tensor cores, with the module API of
h3_sparse_attention/fp8_linear.py (`quantize_rows`, `quantize_tensor`, `swiglu_quantize`,
`swiglu_quantize_tensor`, `Fp8Linear`, `forward_qkv_shared`, `Fp8SwiGLUFeedForward`,
`Fp8AttnProcessor`, `convert_linear_to_fp8`, `install_fp8`), and a finer granularity beside it:
one scale per token and 128 columns of the activation, one per 128 x 128 block of the weight
(`quantize_blocks`, `swiglu_quantize_blocks`, `gelu_quantize_blocks`, `add_rms_norm_quantize`,
`fp8_gemm_blocks`, `Fp8BlockLinear`; `install_fp8(..., scales="block")`).

Scale granularity is per-token activation x per-output-channel weight on every card: the
tcgen05 GEMM in libsparkh3b200.so applies both scale vectors in its epilogue, so the
reference's sm100 switch to per-tensor scales (fp8_linear.py:50-62, 147-156, which exists
only because the library's rowwise-scaled GEMM was slow there) has nothing to buy here.
The per-tensor quantisers stay available and the GEMM accepts a one-element scale on
either side.

Weights are quantised once, at conversion, with the reference's own per-channel recipe
(fp8_linear.py:269-278): scale = max(absmax_row / 448, 1e-12) in fp32, codes =
e4m3(weight / bf16(scale)).  That one-time setup runs as plain torch on whatever device
holds the weight; every per-call operation (activation quantisation, SwiGLU fusion, GEMM)
runs in the CUDA library and fails loudly without it.
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _lib
from .ops import _dtype_code, _require_cuda, _stream

FP8_DTYPE = torch.float8_e4m3fn
FP8_MAX = 448.0
MIN_WIDTH = 4096
SKIP_END_BLOCKS = 0
BLOCK = 128  # columns (and weight rows) per scale of the block-scaled operators


def _rows(x: torch.Tensor) -> torch.Tensor:
    if x.dim() != 2:
        raise ValueError(f"expected [M, K], got {tuple(x.shape)}")
    return x.contiguous()


def quantize_rows(x: torch.Tensor):
    """bf16/fp32 [M, K] -> (e4m3 [M, K], fp32 scale [M, 1]): one absmax per row
    (fp8_linear.py:118-125)."""
    x = _rows(x)
    device = _require_cuda(x)
    M, K = x.shape
    y = torch.empty((M, K), device=device, dtype=FP8_DTYPE)
    scale = torch.empty((M, 1), device=device, dtype=torch.float32)
    with torch.cuda.device(device):
        _lib.call("sb_fp8_quantize_rows", x.data_ptr(), _dtype_code(x), M, K, y.data_ptr(), scale.data_ptr(),
                  _stream(device))
    return y, scale


def quantize_rows_reference(x: torch.Tensor):
    """The eager spelling of quantize_rows (fp8_linear.py:141-144), for the tests."""
    scale = (x.float().abs().amax(dim=1, keepdim=True) / FP8_MAX).clamp_min(1e-12)
    return (x.float() / scale).to(FP8_DTYPE), scale


def swiglu_quantize(h: torch.Tensor):
    """[M, 2K] projection output -> quantize_rows(a * silu(gate)) with a, gate = h.chunk(2),
    without writing the activation (fp8_linear.py:128-138)."""
    h = _rows(h)
    device = _require_cuda(h)
    M, K2 = h.shape
    K = K2 // 2
    y = torch.empty((M, K), device=device, dtype=FP8_DTYPE)
    scale = torch.empty((M, 1), device=device, dtype=torch.float32)
    with torch.cuda.device(device):
        _lib.call("sb_fp8_swiglu_quantize_rows", h.data_ptr(), _dtype_code(h), M, K, y.data_ptr(), scale.data_ptr(),
                  _stream(device))
    return y, scale


def quantize_tensor(x: torch.Tensor):
    """bf16/fp32 [M, K] -> (e4m3 [M, K], fp32 scale [1, 1]): one absmax for the tensor, the
    scale never leaves the device (fp8_linear.py:201-214)."""
    x = _rows(x)
    device = _require_cuda(x)
    y = torch.empty(x.shape, device=device, dtype=FP8_DTYPE)
    scale = torch.empty((1, 1), device=device, dtype=torch.float32)
    workspace = torch.empty(1, device=device, dtype=torch.float32)
    with torch.cuda.device(device):
        _lib.call("sb_fp8_quantize_tensor", x.data_ptr(), _dtype_code(x), x.numel(), y.data_ptr(), scale.data_ptr(),
                  workspace.data_ptr(), _stream(device))
    return y, scale


def quantize_tensor_reference(x: torch.Tensor):
    """The eager spelling of quantize_tensor (fp8_linear.py:217-220), for the tests."""
    scale = (x.float().abs().amax() / FP8_MAX).clamp_min(1e-12).reshape(1, 1)
    return (x.float() / scale).to(FP8_DTYPE), scale


def swiglu_quantize_tensor(h: torch.Tensor):
    """[M, 2K] projection output -> per-tensor quantised bf16(a * silu(gate))
    (fp8_linear.py:223-239)."""
    h = _rows(h)
    device = _require_cuda(h)
    M, K2 = h.shape
    act = torch.empty((M, K2 // 2), device=device, dtype=torch.bfloat16)
    with torch.cuda.device(device):
        _lib.call("sb_fp8_swiglu", h.data_ptr(), _dtype_code(h), M, K2 // 2, act.data_ptr(), _stream(device))
    return quantize_tensor(act)


# ---------------------------------------------------------------- block scales
def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _strided_rows(x: torch.Tensor, name: str) -> tuple[torch.Tensor, int, int, int]:
    """x [M, C] with unit-stride, non-overlapping rows (copied when it has none), M, C and the
    distance between its rows."""
    if x.dim() != 2:
        raise ValueError(f"{name} must be [M, K], got {tuple(x.shape)}")
    if not x.is_cuda:
        raise RuntimeError("spark_h3_b200 kernels require CUDA tensors; there is no CPU path")
    M, C = x.shape
    if C == 0:
        raise ValueError(f"{name} has no columns")
    if x.is_contiguous():
        return x, M, C, C
    stride, unit = x.stride()
    if unit != 1 or (M > 1 and stride < C):
        x, stride = x.contiguous(), C
    return x, M, C, stride if M > 1 else C


def _same_device(index: int, *tensors) -> None:
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise RuntimeError(f"all tensors must be on the same CUDA device: one is on {t.device}, not cuda:{index}")


def _refuse_overlap(out: torch.Tensor, in_place: dict, **inputs) -> None:
    """An output may be one of `in_place` itself, laid out alike: each thread reads those at the
    places that it writes, before it writes them.  Beyond that it overlaps no input, since other
    threads still read it after the first have written."""
    first, last = out.data_ptr(), out.data_ptr() + out.numel() * out.element_size()
    for name, t in {**in_place, **inputs}.items():
        if t is None or t.numel() == 0 or out.numel() == 0:
            continue
        if name in in_place and (t.data_ptr() == first and t.dtype == out.dtype and t.shape == out.shape
                                 and t.is_contiguous()):
            continue
        span = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1
        if t.data_ptr() < last and first < t.data_ptr() + span * t.element_size():
            raise ValueError(f"out overlaps {name}" + (" without being it" if name in in_place else ""))


def _call_on(index: int, name: str, *args) -> None:
    """The C-ABI call with CUDA device `index` current, on its current stream.  These operators take
    a few microseconds on a few rows, so the host side keeps to the cheapest forms of its queries."""
    fn = _lib.bound(name)
    if torch._C._cuda_getDevice() == index:
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if status < 0:
        _lib.check(status, name)


def _quantize_blocks(entry: str, x: torch.Tensor, halves: int):
    x, M, K, stride = _strided_rows(x, "x")
    dtype = _dtype_code(x)
    if halves != 1:
        if K % halves:
            raise ValueError(f"a [M, 2K] projection output is expected, got {tuple(x.shape)}")
        K //= halves
    device = x.device
    y = torch.empty(M, K, device=device, dtype=FP8_DTYPE)
    scale = torch.empty(M, -(-K // BLOCK), device=device, dtype=torch.float32)
    if M > 0:
        _call_on(device.index, entry, x.data_ptr(), stride, dtype, M, K, y.data_ptr(), scale.data_ptr())
    return y, scale


def quantize_blocks(x: torch.Tensor):
    """bf16/fp32 [M, K] -> (e4m3 [M, K], fp32 scales [M, ceil(K / 128)]): one absmax per row and
    128 columns.  Rows may be strided (a column slice is read in place)."""
    return _quantize_blocks("sb_fp8_quantize_blocks", x, 1)


def quantize_blocks_reference(x: torch.Tensor):
    """The eager spelling of quantize_blocks, for the tests."""
    M, K = x.shape
    y = F.pad(x.float(), (0, _blocks(K) * BLOCK - K)).view(M, -1, BLOCK)
    scale = (y.abs().amax(dim=2) / FP8_MAX).clamp_min(1e-12)
    return (y / scale[:, :, None]).to(FP8_DTYPE).view(M, -1)[:, :K], scale


def swiglu_quantize_blocks(h: torch.Tensor):
    """[M, 2K] projection output -> quantize_blocks(a * silu(gate)) with a, gate = h.chunk(2),
    without writing the activation."""
    return _quantize_blocks("sb_fp8_swiglu_quantize_blocks", h, 2)


def gelu_quantize_blocks(x: torch.Tensor):
    """quantize_blocks(gelu(x)) (erf form) without writing the activation."""
    return _quantize_blocks("sb_fp8_gelu_quantize_blocks", x, 1)


def _sample_vector(v: torch.Tensor, name: str, M: int, C: int, samples: int):
    """A vector [C] or one per sample [S, C] as (fp32 tensor, stride between samples, S)."""
    shape = v.shape
    if shape[-1:] != (C,) or len(shape) > 2:
        raise ValueError(f"{name} must be [{C}] or [samples, {C}], got {tuple(shape)}")
    if v.dtype != torch.float32:
        v = v.float()
    if not v.is_contiguous() and v.stride(-1) != 1:
        v = v.contiguous()
    if len(shape) == 1 or shape[0] == 1:
        return v, 0, samples
    S = shape[0]
    if S == 0 or M % S or (samples not in (1, S)):
        raise ValueError(f"{name} has {S} samples: {M} rows must split evenly among one number of samples")
    return v, v.stride(0), S


def add_rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None, *,
                          gate: torch.Tensor | None = None, shift: torch.Tensor | None = None, eps: float = 1e-6,
                          blocks: bool = True, out: torch.Tensor | None = None):
    """s = residual + gate * x; y = s * rsqrt(mean(s^2) + eps) * weight + shift; y in e4m3.

    x, residual: bf16/fp32 [M, C], C <= 16384, rows may be strided.  weight, gate, shift: [C],
    or [S, C] with one row per sample (S divides M; row m belongs to sample m // (M / S)).
    Returns (codes [M, C], scales, s): scales [M, ceil(C / 128)] (`blocks`, for fp8_gemm_blocks)
    or [M, 1] (for fp8_gemm); s in x's dtype, written to `out` when given (which may be the
    residual itself, the residual stream updated in place, or x, and overlaps no other input), or
    None without a residual.  The norm works on the unrounded fp32 sum.  Outputs carry no gradient."""
    x, M, C, x_stride = _strided_rows(x, "x")
    device, dtype = x.device, _dtype_code(x)
    r_stride, residual_ptr, out_ptr = 0, None, None
    if residual is None:
        if gate is not None or out is not None:
            raise ValueError("gate and out belong to the residual's addition: pass a residual")
    else:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"the residual must match x: {tuple(residual.shape)} {residual.dtype}, "
                             f"not {tuple(x.shape)} {x.dtype}")
        residual, _, _, r_stride = _strided_rows(residual, "residual")
        if out is None:
            out = torch.empty(M, C, device=device, dtype=x.dtype)
        elif out.shape != x.shape or out.dtype != x.dtype or not out.is_contiguous():
            raise ValueError(f"out must be contiguous {tuple(x.shape)} {x.dtype}")
        else:
            _refuse_overlap(out, dict(x=x, residual=residual), weight=weight, gate=gate, shift=shift)
        residual_ptr, out_ptr = residual.data_ptr(), out.data_ptr()
    _same_device(device.index, residual, weight, gate, shift, out)
    samples, gate_ptr, g_stride, weight_ptr, w_stride, shift_ptr, s_stride = 1, None, 0, None, 0, None, 0
    if gate is not None:
        gate, g_stride, samples = _sample_vector(gate, "gate", M, C, samples)
        gate_ptr = gate.data_ptr()
    if weight is not None:
        weight, w_stride, samples = _sample_vector(weight, "weight", M, C, samples)
        weight_ptr = weight.data_ptr()
    if shift is not None:
        shift, s_stride, samples = _sample_vector(shift, "shift", M, C, samples)
        shift_ptr = shift.data_ptr()
    y = torch.empty(M, C, device=device, dtype=FP8_DTYPE)
    scale = torch.empty(M, _blocks(C) if blocks else 1, device=device, dtype=torch.float32)
    if M > 0:
        _call_on(device.index, "sb_fp8_add_rms_norm_quantize", x.data_ptr(), x_stride, residual_ptr, r_stride, gate_ptr,
                 g_stride, weight_ptr, w_stride, shift_ptr, s_stride, dtype, M, C, M // samples, eps, 1 if blocks else 0,
                 out_ptr, y.data_ptr(), scale.data_ptr())
    return y, scale, out


def fp8_gemm_blocks(a_fp8: torch.Tensor, a_scale: torch.Tensor, b_fp8: torch.Tensor, b_scale: torch.Tensor,
                    bias: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
                    gate: torch.Tensor | None = None, out: torch.Tensor | None = None,
                    out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """[M, N] = a_fp8 [M, K] . b_fp8 [N, K]^T with a_scale [M, ceil(K / 128)] (any strides) applied
    per row and 128 columns and b_scale [ceil(N / 128), ceil(K / 128)] per 128 x 128 block
    (+ bias [N]); residual + gate * (that) with a residual [M, N] of the output's dtype (gate [N],
    1 when None).  out_dtype bf16 (the default) or fp32; `out` may be the residual itself and overlaps
    no other input.  K must be a multiple of 16; the operands, the residual and `out` start on 16
    bytes.  The output carries no gradient."""
    if a_fp8.dtype != FP8_DTYPE or b_fp8.dtype != FP8_DTYPE:
        raise TypeError("fp8_gemm_blocks takes float8_e4m3fn operands")
    if a_fp8.dim() != 2 or b_fp8.dim() != 2 or a_fp8.shape[1] != b_fp8.shape[1]:
        raise ValueError(f"A [M, K] and B [N, K] must share K: {tuple(a_fp8.shape)} vs {tuple(b_fp8.shape)}")
    if not a_fp8.is_cuda:
        raise RuntimeError("spark_h3_b200 kernels require CUDA tensors; there is no CPU path")
    index = a_fp8.get_device()
    _same_device(index, a_scale, b_fp8, b_scale)
    (M, K), N = a_fp8.shape, b_fp8.shape[0]
    if a_scale.dtype != torch.float32 or b_scale.dtype != torch.float32:
        raise TypeError(f"{'b' if a_scale.dtype == torch.float32 else 'a'}_scale must be float32")
    kb = -(-K // BLOCK)
    if a_scale.shape != (M, kb):
        raise ValueError(f"a_scale must be [{M}, {kb}], got {tuple(a_scale.shape)}")
    if b_scale.shape != (-(-N // BLOCK), kb):
        raise ValueError(f"b_scale must be [{_blocks(N)}, {kb}], got {tuple(b_scale.shape)}")
    a_fp8, b_fp8, b_scale = a_fp8.contiguous(), b_fp8.contiguous(), b_scale.contiguous()
    if out_dtype is None:
        out_dtype = torch.bfloat16 if out is None else out.dtype
    if out is None:
        out = torch.empty(M, N, device=a_fp8.device, dtype=out_dtype)
    else:
        if out.shape != (M, N) or out.dtype != out_dtype or not out.is_contiguous():
            raise ValueError(f"out must be contiguous [{M}, {N}] {out_dtype}")
        _same_device(index, out)
        _refuse_overlap(out, dict(residual=residual), a_fp8=a_fp8, a_scale=a_scale, b_fp8=b_fp8, b_scale=b_scale,
                        bias=bias, gate=gate)
    code = _dtype_code(out)
    bias_ptr = residual_ptr = gate_ptr = None
    if bias is not None:
        _same_device(index, bias)
        bias = bias.float().contiguous()
        if bias.numel() != N:
            raise ValueError(f"bias needs {N} values, got {bias.numel()}")
        bias_ptr = bias.data_ptr()
    if residual is not None:
        if residual.shape != (M, N) or residual.dtype != out_dtype:
            raise ValueError(f"the residual must be [{M}, {N}] {out_dtype}")
        _same_device(index, residual, gate)
        residual = residual.contiguous()
        residual_ptr = residual.data_ptr()
        if gate is not None:
            gate = gate.float().contiguous()
            if gate.numel() != N:
                raise ValueError(f"gate needs {N} values, got {gate.numel()}")
            gate_ptr = gate.data_ptr()
    elif gate is not None:
        raise ValueError("gate belongs to the residual's addition: pass a residual")
    if M > 0 and N > 0:
        row_stride, block_stride = a_scale.stride()
        _call_on(index, "sb_fp8_gemm_blocks", a_fp8.data_ptr(), a_scale.data_ptr(), row_stride, block_stride,
                 b_fp8.data_ptr(), b_scale.data_ptr(), M, N, K, bias_ptr, residual_ptr, gate_ptr, out.data_ptr(), code)
    return out


def quantize_weight_blocks(weight: torch.Tensor):
    """e4m3 weight with one scale per 128 x 128 block: (codes [N, K], scales [ceil(N / 128),
    ceil(K / 128)]), scale = max(absmax / 448, 1e-12) in fp32, codes = e4m3(weight / scale)."""
    if weight.dim() != 2:
        raise ValueError(f"expected a weight [N, K], got {tuple(weight.shape)}")
    N, K = weight.shape
    w = F.pad(weight.float(), (0, _blocks(K) * BLOCK - K, 0, _blocks(N) * BLOCK - N))
    w = w.view(_blocks(N), BLOCK, _blocks(K), BLOCK)
    scale = (w.abs().amax(dim=(1, 3)) / FP8_MAX).clamp_min(1e-12)
    codes = (w / scale[:, None, :, None]).to(FP8_DTYPE).view(_blocks(N) * BLOCK, -1)
    return codes[:N, :K].contiguous(), scale


def quantize_activation(x: torch.Tensor):
    """What the GEMM callers use: per-token scales (the GEMM epilogue applies them)."""
    return quantize_rows(x)


def swiglu_quantize_activation(h: torch.Tensor):
    return swiglu_quantize(h)


def fp8_gemm(a_fp8: torch.Tensor, a_scale: torch.Tensor, b_fp8: torch.Tensor, b_scale: torch.Tensor,
             bias: torch.Tensor | None = None, out: torch.Tensor | None = None, num_ctas: int = 0) -> torch.Tensor:
    """bf16 [M, N] = (a_fp8 [M, K] . b_fp8 [N, K]^T) * a_scale * b_scale (+ bias).  Each scale
    holds one value per row of its operand, or a single value for the whole operand."""
    a_fp8, b_fp8 = a_fp8.contiguous(), b_fp8.contiguous()
    device = _require_cuda(a_fp8, b_fp8, a_scale.contiguous(), b_scale.contiguous(), bias, out)
    if a_fp8.dtype != FP8_DTYPE or b_fp8.dtype != FP8_DTYPE:
        raise TypeError("fp8_gemm takes float8_e4m3fn operands")
    M, K = a_fp8.shape
    N = b_fp8.shape[0]
    if b_fp8.shape[1] != K:
        raise ValueError(f"A [M, K] and B [N, K] must share K: {tuple(a_fp8.shape)} vs {tuple(b_fp8.shape)}")
    scales = []
    for scale, rows, name in ((a_scale, M, "a_scale"), (b_scale, N, "b_scale")):
        if scale.dtype != torch.float32:
            raise TypeError(f"{name} must be float32")
        if scale.numel() not in (1, rows):
            raise ValueError(f"{name} needs 1 or {rows} values, got {scale.numel()}")
        scales.append((scale.contiguous(), 1 if scale.numel() == rows and rows > 1 else 0))
    (a_scale, a_stride), (b_scale, b_stride) = scales
    if bias is not None:
        bias = bias.to(torch.bfloat16).contiguous()
        if bias.numel() != N:
            raise ValueError(f"bias needs {N} values, got {bias.numel()}")
    if out is None:
        out = torch.empty((M, N), device=device, dtype=torch.bfloat16)
    with torch.cuda.device(device):
        _lib.call("sb_fp8_gemm", a_fp8.data_ptr(), a_scale.data_ptr(), a_stride, b_fp8.data_ptr(), b_scale.data_ptr(),
                  b_stride, M, N, K, None if bias is None else bias.data_ptr(), out.data_ptr(), num_ctas,
                  _stream(device))
    return out


def quantize_weight(weight: torch.Tensor):
    """Per-output-channel e4m3 weight (fp8_linear.py:269-278): (codes [N, K], scale [1, N])."""
    scale = (weight.abs().amax(dim=1, keepdim=True).float() / FP8_MAX).clamp_min(1e-12)
    codes = (weight / scale.to(weight.dtype)).to(FP8_DTYPE)
    return codes, scale.reshape(1, -1).contiguous()


class Fp8Linear(nn.Module):
    """A bias-optional Linear whose GEMM runs in e4m3 on the tensor cores (fp8_linear.py:252-293).

    The weight is quantised once, per output channel; the activation is quantised per token
    on every call, or by the caller (`forward_quantized`) when one activation feeds several
    of these.  Only the e4m3 copy, its scales and the bias are kept."""

    def __init__(self, linear: nn.Linear):
        super().__init__()
        codes, scale = quantize_weight(linear.weight.detach())
        self.register_buffer("weight_fp8", codes)
        self.register_buffer("weight_scale", scale)
        self.register_parameter("bias", linear.bias)
        self.in_features = linear.in_features
        self.out_features = linear.out_features

    def forward_quantized(self, x_fp8, x_scale, out_dtype=torch.bfloat16):
        """[M, K] e4m3 rows and their scales ([M, 1] per token or [1, 1]) -> [M, N]."""
        bias = None if self.bias is None else self.bias.detach()
        out = fp8_gemm(x_fp8, x_scale, self.weight_fp8, self.weight_scale, bias)
        return out if out_dtype == torch.bfloat16 else out.to(out_dtype)

    # the activation quantisers whose scales this linear's GEMM takes
    quantize = staticmethod(quantize_activation)
    swiglu_quantize = staticmethod(swiglu_quantize_activation)

    def forward(self, x):
        shape = x.shape
        rows = x.reshape(-1, shape[-1])
        out = self.forward_quantized(*self.quantize(rows), out_dtype=rows.dtype)
        return out.reshape(*shape[:-1], self.out_features)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


class Fp8BlockLinear(Fp8Linear):
    """Fp8Linear with block scales: one per token and 128 columns of the activation, one per
    128 x 128 block of the weight.  A large value then pushes only its own block's small values
    into e4m3's subnormals.  Inference only, like Fp8Linear; in_features must be a multiple of 16."""

    def __init__(self, linear: nn.Linear):
        nn.Module.__init__(self)
        if linear.in_features % 16:
            raise ValueError(f"Fp8BlockLinear needs in_features in multiples of 16, got {linear.in_features}")
        codes, scale = quantize_weight_blocks(linear.weight.detach())
        self.register_buffer("weight_fp8", codes)
        self.register_buffer("weight_scale", scale)
        self.register_parameter("bias", linear.bias)
        self.in_features = linear.in_features
        self.out_features = linear.out_features

    quantize = staticmethod(quantize_blocks)
    swiglu_quantize = staticmethod(swiglu_quantize_blocks)

    def forward_quantized(self, x_fp8, x_scale, out_dtype=torch.bfloat16):
        """[M, K] e4m3 rows and their scales [M, ceil(K / 128)] -> [M, N]."""
        bias = None if self.bias is None else self.bias.detach()
        kernel_dtype = torch.float32 if out_dtype == torch.float32 else torch.bfloat16
        out = fp8_gemm_blocks(x_fp8, x_scale, self.weight_fp8, self.weight_scale, bias, out_dtype=kernel_dtype)
        return out if out_dtype == kernel_dtype else out.to(out_dtype)


def forward_qkv_shared(attn, hidden_states):
    """One quantisation of hidden_states feeds q/k/v when all three are Fp8Linear of one scale
    granularity (fp8_linear.py:296-310); None otherwise, and the caller runs the plain
    projections."""
    projections = (attn.to_q, attn.to_k, attn.to_v)
    if not all(isinstance(p, Fp8Linear) and p.quantize is projections[0].quantize for p in projections):
        return None
    rows = hidden_states.reshape(-1, hidden_states.shape[-1])
    x_fp8, x_scale = attn.to_q.quantize(rows)
    return tuple(p.forward_quantized(x_fp8, x_scale, out_dtype=hidden_states.dtype)
                 .reshape(*hidden_states.shape[:-1], p.out_features) for p in projections)


class Fp8SwiGLUFeedForward(nn.Module):
    """FeedForward([SwiGLU, Dropout(0), Linear]) with both GEMMs in e4m3 and the SwiGLU fused
    into the quantisation of its output (fp8_linear.py:313-336); inference only."""

    def __init__(self, ff):
        super().__init__()
        swiglu, dropout, down = ff.net
        if getattr(dropout, "p", 0) != 0:
            raise ValueError("Fp8SwiGLUFeedForward fuses the activation with the quantisation; a live dropout "
                             "cannot be fused")
        self.proj = swiglu.proj
        self.down = down

    def forward(self, hidden_states):
        shape = hidden_states.shape
        h = self.proj(hidden_states.reshape(-1, shape[-1]))
        out = self.down.forward_quantized(*self.down.swiglu_quantize(h), out_dtype=h.dtype)
        return out.reshape(*shape[:-1], self.down.out_features)


class Fp8AttnProcessor:
    """Dense attention processor with one quantisation of hidden_states shared by q/k/v
    (fp8_linear.py:339-379).  Installed by `install_fp8` where all three projections are
    Fp8Linear; the sparse plugin adopts it as its dense path when installed afterwards."""

    _attention_backend = None
    _parallel_config = None

    def __call__(self, attn, hidden_states, rotary_emb=None, attention_mask=None):
        from .processor import apply_rotary_emb

        projected = forward_qkv_shared(attn, hidden_states)
        if projected is None:  # projections replaced since, or of different granularity
            projected = (attn.to_q(hidden_states), attn.to_k(hidden_states), attn.to_v(hidden_states))
        query, key, value = projected
        query = attn.norm_q(query.unflatten(-1, (attn.heads, -1)))
        key = attn.norm_k(key.unflatten(-1, (attn.heads, -1)))
        value = value.unflatten(-1, (attn.heads, -1))
        if rotary_emb is not None:
            query = apply_rotary_emb(query, rotary_emb)
            key = apply_rotary_emb(key, rotary_emb)
        out = F.scaled_dot_product_attention(query.transpose(1, 2), key.transpose(1, 2), value.transpose(1, 2),
                                             attn_mask=attention_mask)
        hidden_states = out.transpose(1, 2).flatten(2, 3).type_as(query)
        hidden_states = attn.to_out[0](hidden_states)
        return attn.to_out[1](hidden_states)


def _fuse_ff(block) -> bool:
    """block.ff -> Fp8SwiGLUFeedForward when both of its GEMMs became Fp8Linear
    (fp8_linear.py:382-395)."""
    ff = getattr(block, "ff", None)
    net = getattr(ff, "net", None)
    if net is None or len(net) != 3:
        return False
    swiglu, dropout, down = net
    if not (isinstance(getattr(swiglu, "proj", None), Fp8Linear) and isinstance(down, Fp8Linear)
            and getattr(dropout, "p", 0) == 0):
        return False
    block.ff = Fp8SwiGLUFeedForward(ff)
    return True


def convert_linear_to_fp8(model, min_width=MIN_WIDTH, skip_end_blocks=SKIP_END_BLOCKS, scales="channel"):
    """Swap the Linears at least `min_width` wide on both sides inside
    model.transformer_blocks for Fp8Linear, in place, and fuse each converted block's SwiGLU
    FeedForward (fp8_linear.py:398-427).  `skip_end_blocks` keeps the first and last N blocks
    in bf16.  `scales`: "channel" (per token x per output channel, Fp8Linear) or "block" (per
    128 columns x per 128 x 128 block, Fp8BlockLinear; Linears whose in_features is no multiple of
    16 stay as they are).  Returns how many Linears were swapped."""
    if scales not in ("channel", "block"):
        raise ValueError(f'scales must be "channel" or "block", got {scales!r}')
    kind = Fp8Linear if scales == "channel" else Fp8BlockLinear
    blocks = getattr(model, "transformer_blocks", None)
    if not blocks:
        raise ValueError("convert_linear_to_fp8 expects a model with a non-empty `transformer_blocks` ModuleList")
    swapped = 0
    for index, block in enumerate(blocks):
        if index < skip_end_blocks or index >= len(blocks) - skip_end_blocks:
            continue
        for parent in list(block.modules()):
            for name, child in list(parent.named_children()):
                if not isinstance(child, nn.Linear):
                    continue
                if child.in_features < min_width or child.out_features < min_width:
                    continue
                if kind is Fp8BlockLinear and child.in_features % 16:
                    continue
                setattr(parent, name, kind(child).to(child.weight.device))
                swapped += 1
        _fuse_ff(block)
    return swapped


def install_fp8(pipe_or_transformer, min_width=MIN_WIDTH, skip_end_blocks=SKIP_END_BLOCKS, scales="channel"):
    """Convert a pipeline's (or a transformer's) wide block Linears, fuse the FeedForwards and
    install the shared-qkv processor on every converted attention (fp8_linear.py:430-447).
    Call after the weights are loaded and before the sparse-attention plugin.  `scales` is the
    granularity of convert_linear_to_fp8.  Returns how many Linears were quantised."""
    transformer = getattr(pipe_or_transformer, "transformer", pipe_or_transformer)
    swapped = convert_linear_to_fp8(transformer, min_width=min_width, skip_end_blocks=skip_end_blocks, scales=scales)
    for block in transformer.transformer_blocks:
        attn = getattr(block, "attn", None)
        if (attn is not None and not getattr(attn, "fused_projections", False)
                and all(isinstance(getattr(attn, name, None), Fp8Linear) for name in ("to_q", "to_k", "to_v"))):
            attn.set_processor(Fp8AttnProcessor())
    return swapped
