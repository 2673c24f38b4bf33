"""Block-scaled e4m3 operators (one scale per row and 128 columns, one per 128 x 128 weight block)
against their definition in 64 bits.

Tolerances.  A code is the nearest e4m3 value of y / scale, where the kernel's quotient may be off
by `slack` of itself: 2^-22 from the reciprocal (2^-23) and the product (2^-24), plus the error of the
fp32 y.
A GEMM sums blocks of 128 exact products in fp32: each of the 128 + blocks additions rounds (or
truncates) to at most 2^-23 of the sum of the terms' magnitudes; its output then rounds once
(eps / 2 of the value)."""
from __future__ import annotations

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from spark_h3_b200 import _lib, fp8_linear as fl, ops

E4M3 = torch.float8_e4m3fn
_P = 0x10000  # a non-null, 16-byte aligned address that validation never dereferences


def blocks_of(n):
    return -(-n // 128)


def spread(scale, K):
    return scale.repeat_interleave(128, dim=1)[:, :K]


def group_absmax(y):
    M, K = y.shape
    return F.pad(y, (0, blocks_of(K) * 128 - K)).view(M, -1, 128).abs().amax(dim=2)


def assert_nearest_codes(codes, quotient, slack):
    """Each code is an e4m3 value nearest to a value within slack * |quotient| (a tensor or a
    number) of the quotient (fp64)."""
    got = codes.double()
    q = quotient.clamp(-448, 448)
    exponent = torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -40))).clamp_min(-6)
    half_step = torch.exp2(exponent - 4)
    # at a binade's edge the nearest value may lie in the next binade: its half step is twice
    off = (got - q).abs() - half_step * (1 + 1e-12) - 2 * slack * q.abs()
    assert bool((off <= 0).all()), float(off.max())


def special(x):
    """Scatter the type's extreme values over some groups of x."""
    x = x.clone()
    x[0, 3] = float("nan")
    x[-1, -1] = float("inf")
    x[x.shape[0] // 2, :] = 0
    return x


# ------------------------------------------------------------------------------ CPU: refusals

def test_cpu_tensors_are_refused():
    x = torch.randn(4, 256)
    for call in (lambda: fl.quantize_blocks(x), lambda: fl.swiglu_quantize_blocks(x), lambda: fl.gelu_quantize_blocks(x),
                 lambda: fl.add_rms_norm_quantize(x),
                 lambda: fl.fp8_gemm_blocks(x.to(E4M3), torch.ones(4, 2), x.to(E4M3), torch.ones(1, 2))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match=r"\[M, K\]"):
        fl.quantize_blocks(torch.randn(4))


_NORM = dict(x=_P, x_stride=256, residual=_P, residual_stride=256, gate=_P, gate_stride=0, weight=_P, weight_stride=0,
             shift=_P, shift_stride=0, dtype=1, M=4, C=256, rows=4, eps=1e-6, blocks=1, summed=_P, out=_P, scales=_P,
             stream=None)


@pytest.mark.parametrize("change,message,code", [
    (dict(x=None), "null pointer", -1), (dict(out=None), "null pointer", -1), (dict(dtype=5), "bad dtype", -1),
    (dict(M=0), "M in [1, 2^31)", -1), (dict(M=1 << 31), "M in [1, 2^31)", -1), (dict(C=0), "C positive", -1),
    (dict(summed=None), "come together", -1), (dict(residual=None), "come together", -1),
    (dict(residual=None, summed=None), "a gate needs a residual", -1), (dict(x_stride=255), "rows overlap", -1),
    (dict(residual_stride=0), "rows overlap", -1), (dict(rows=0), "whole number of samples", -1),
    (dict(rows=3), "whole number of samples", -1), (dict(blocks=2), "blocks must be 0 or 1", -1),
    (dict(x=_P + 1), "aligned to their elements", -1), (dict(scales=_P + 2), "aligned to their elements", -1),
    (dict(shift_stride=-1), "must not be negative", -1), (dict(C=16385, x_stride=20000, residual_stride=20000), "at most 16384 columns", -3)])
def test_norm_rejects_bad_arguments(change, message, code):
    lib = _lib.load()
    assert lib.sb_fp8_add_rms_norm_quantize(*{**_NORM, **change}.values()) == code
    assert message in lib.sb_last_error().decode()


@pytest.mark.parametrize("entry,halves", [("sb_fp8_quantize_blocks", 1), ("sb_fp8_swiglu_quantize_blocks", 2),
                                          ("sb_fp8_gelu_quantize_blocks", 1)])
def test_quantisers_reject_bad_arguments(entry, halves):
    lib = _lib.load()
    valid = dict(x=_P, stride=256 * halves, dtype=1, M=4, K=256, out=_P, scales=_P, stream=None)
    for change, message in ((dict(x=None), "null pointer"), (dict(scales=None), "null pointer"),
                            (dict(dtype=2), "bad dtype"), (dict(M=0), "M in [1, 2^31)"), (dict(K=0), "K in [1, 2^24]"),
                            (dict(stride=256 * halves - 1), "rows overlap"), (dict(x=_P + 1), "aligned to their elements"),
                            (dict(scales=_P + 2), "aligned to their elements")):
        assert getattr(lib, entry)(*{**valid, **change}.values()) == -1, change
        assert entry in lib.sb_last_error().decode() and message in lib.sb_last_error().decode()


def test_gemm_rejects_bad_arguments():
    lib = _lib.load()
    valid = dict(a=_P, a_scale=_P, rs=2, bs=1, b=_P, b_scale=_P, M=4, N=64, K=256, bias=None, residual=None, gate=None,
                 out=_P, dtype=1, stream=None)
    for change, message in ((dict(a=None), "null pointer"), (dict(out=None), "null pointer"),
                            (dict(dtype=3), "bad output dtype"), (dict(M=0), "must be positive"),
                            (dict(N=-1), "must be positive"), (dict(K=0), "must be positive"),
                            (dict(M=1 << 31), "at most 2^31 - 256"), (dict(K=250), "multiple of 16"),
                            (dict(a=_P + 8), "16-byte aligned"), (dict(out=_P + 4), "16-byte aligned"),
                            (dict(residual=_P + 2), "16-byte aligned"), (dict(bias=_P + 2), "4-byte aligned"),
                            (dict(gate=_P), "a gate needs a residual"), (dict(rs=-1), "must not be negative")):
        assert lib.sb_fp8_gemm_blocks(*{**valid, **change}.values()) == -1, change
        assert message in lib.sb_last_error().decode(), (change, lib.sb_last_error())


def test_weight_blocks_follow_their_definition():
    torch.manual_seed(3)
    w = (torch.randn(200, 300) * 0.02).to(torch.bfloat16)
    w[:128, 128:256] = 0
    codes, scale = fl.quantize_weight_blocks(w)
    assert codes.shape == w.shape and codes.dtype == E4M3 and scale.shape == (2, 3)
    for nb in range(2):
        for kb in range(3):
            block = w[nb * 128:(nb + 1) * 128, kb * 128:(kb + 1) * 128].float()
            s = (block.abs().max() / 448).clamp_min(1e-12)
            assert scale[nb, kb] == s
            assert torch.equal(codes[nb * 128:(nb + 1) * 128, kb * 128:(kb + 1) * 128].view(torch.uint8),
                               (block / s).to(E4M3).view(torch.uint8))


def test_block_scales_install_scope():
    from test_fp8_linear import FeedForward, fake_model

    model = fake_model()
    assert fl.convert_linear_to_fp8(model, min_width=8, skip_end_blocks=2, scales="block") == 6
    assert type(model.transformer_blocks[4].wide) is fl.Fp8BlockLinear
    with pytest.raises(ValueError, match="channel"):
        fl.install_fp8(fake_model(), min_width=8, scales="tensor")
    with pytest.raises(ValueError, match="multiples of 16"):
        fl.Fp8BlockLinear(nn.Linear(24, 16))
    block = nn.Module()
    block.ff = FeedForward()
    model = nn.Module()
    model.transformer_blocks = nn.ModuleList([block])
    fl.convert_linear_to_fp8(model, min_width=8, scales="block")
    assert type(block.ff) is fl.Fp8SwiGLUFeedForward and type(block.ff.down) is fl.Fp8BlockLinear


# ------------------------------------------------------------------------------ GPU: quantisers

ACTIVATIONS = {
    "none": (fl.quantize_blocks, lambda x: x),
    "swiglu": (fl.swiglu_quantize_blocks, lambda x: x.chunk(2, 1)[0] * x.chunk(2, 1)[1] * torch.sigmoid(x.chunk(2, 1)[1])),
    "gelu": (fl.gelu_quantize_blocks, lambda x: x * torch.special.ndtr(x)),
}


def check_quantised(codes, scale, y, y_error):
    """codes / scale of y (fp64) whose fp32 evaluation is off by at most y_error (tensor)."""
    M, K = y.shape
    assert codes.shape == (M, K) and codes.dtype == E4M3
    assert scale.shape == (M, blocks_of(K)) and scale.dtype == torch.float32
    amax = group_absmax(y)
    want = (amax / 448).clamp_min(1e-12)
    # fp32(1/448) and the product: 2^-23 of the scale, and the largest error of its block
    assert bool(((scale.double() - want).abs() <= want * 2.0 ** -23 + group_absmax(y_error) / 448).all())
    s = spread(scale.double(), K)
    q = y / s
    assert_nearest_codes(codes, q, 2.0 ** -22 + (y_error / s) / q.abs().clamp_min(1e-30))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", ["none", "swiglu", "gelu"])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 129), (5, 1000), (2, 4104), (517, 136), (1, 14336), (67, 8192), (40, 130), (33, 2490)])
def test_quantisers_match_their_definition(cuda_device, dtype, act, M, K):
    g = torch.Generator(device=cuda_device).manual_seed(M * 10007 + K)
    call, formula = ACTIVATIONS[act]
    x = (torch.randn(M, 2 * K if act == "swiglu" else K, device=cuda_device, generator=g) * 3).clamp(-16, 16).to(dtype)
    y = formula(x.double())
    if act == "none":
        error = torch.zeros_like(y)
    elif act == "swiglu":  # exp's argument is off by |g| 2^-23, its value by 2^-22, four more operations by 2^-23 each
        error = y.abs() * (x.chunk(2, 1)[1].double().abs() * 2.0 ** -23 + 2.0 ** -20)
    else:  # 1 + erf is off by 2^-23 in absolute terms beside its own rounding, erf's argument by 2^-23 |x|
        error = x.double().abs() * 2.0 ** -21 + y.abs() * 2.0 ** -22
    check_quantised(*call(x), y, error)
    if act == "none":  # the scale is the eager spelling's, bit for bit
        _, scale = call(x)
        assert torch.equal(scale, (group_absmax(x.float()) * torch.tensor(1 / 448, device=cuda_device)).clamp_min(1e-12))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "swiglu", "gelu"])
def test_quantisers_read_strided_and_misaligned_rows(cuda_device, act):
    call, _ = ACTIVATIONS[act]
    halves = 2 if act == "swiglu" else 1
    base = torch.randn(40, 2100, device=cuda_device, dtype=torch.bfloat16)
    for view in (base[:, 8:8 + 256 * halves], base[:, 3:3 + 200 * halves], base[:, 2:2 + 256 * halves], base[::3, :128 * halves],
                 base.t()[:130, :40 // halves * halves], base[:1].expand(6, 2100), base.view(-1)[5:5 + 32 * 512].view(32, 512)):
        want = call(view.clone(memory_format=torch.contiguous_format))
        got = call(view)
        assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_quantisers_special_values(cuda_device):
    x = special(torch.randn(7, 300, device=cuda_device))
    x[1, 0], x[2, 0] = 3e38, 1e-40
    for dtype in (torch.bfloat16, torch.float32):
        t = x.to(dtype)
        codes, scale = fl.quantize_blocks(t)
        want = (group_absmax(t.float()) * torch.tensor(1 / 448, device=cuda_device)).clamp_min(1e-12)
        assert torch.equal(scale.nan_to_num(-1.0), want.nan_to_num(-1.0))
        assert bool(scale[0, 0].isnan()) and bool(codes[0, :128].float().isnan().all())
        assert not bool(codes[0, 128:].float().isnan().any())
        assert bool(scale[-1, -1].isinf()) and bool(codes[-1, -1].float().isnan())
        assert bool((codes[-1, 256:-1].float() == 0).all())
        assert bool((codes[3].float() == 0).all()) and bool((scale[3] == 1e-12).all())
    for empty in (torch.empty(0, 256, device=cuda_device), torch.empty(0, 256, device=cuda_device, dtype=torch.bfloat16)):
        codes, scale = fl.quantize_blocks(empty)
        assert codes.shape == (0, 256) and scale.shape == (0, 2)


# ------------------------------------------------------------------------------ GPU: norm

def norm_reference(x, weight, residual, gate, shift, eps):
    def rows(v):
        if v is None or v.dim() == 1:
            return v if v is None else v.double()
        return v.double().repeat_interleave(x.shape[0] // v.shape[0], dim=0)

    s = x.double()
    if residual is not None:
        s = residual.double() + (s if gate is None else rows(gate) * s)
    n = s * torch.rsqrt(s.square().mean(dim=1, keepdim=True) + eps)
    y = n if weight is None else n * rows(weight)
    # fp32: the sum, the mean of squares (C roundings of at most half a step each, averaged), rsqrt and two products
    magnitude = y.abs()
    if residual is not None:
        inner = residual.double().abs() + (x.double() if gate is None else rows(gate) * x.double()).abs()
        magnitude = magnitude + (inner * torch.rsqrt(s.square().mean(dim=1, keepdim=True) + eps)
                                 * (1 if weight is None else rows(weight).abs()))
    if shift is not None:
        y = y + rows(shift)
        magnitude = magnitude + y.abs()
    return s, y, magnitude * 2.0 ** -20


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("blocks", [True, False])
@pytest.mark.parametrize("M,C,residual,gate,shift,samples", [
    (1, 4096, True, False, False, 1), (1, 1, False, False, False, 1), (6, 128, True, True, True, 3),
    (259, 5376, True, False, True, 1), (4, 257, True, True, True, 2), (33, 1000, False, False, True, 1),
    (2, 16384, True, True, True, 2), (3, 9911, True, True, False, 1), (700, 1024, True, False, False, 1),
    (9, 2048, False, False, False, 1), (1200, 4096, True, True, True, 2),
    (6, 130, True, True, True, 3), (40, 2490, True, True, True, 2), (3, 12942, True, False, True, 1), (5, 8192, True, True, True, 5)])
def test_add_rms_norm_quantize(cuda_device, dtype, blocks, M, C, residual, gate, shift, samples):
    g = torch.Generator(device=cuda_device).manual_seed(M * 31 + C)

    def rand(*shape):
        return torch.randn(*shape, device=cuda_device, generator=g)

    vec = (samples, C) if samples > 1 else (C,)
    x = (rand(M, C) * 2).to(dtype)
    r = (rand(M, C) * 3).to(dtype) if residual else None
    w, b, t = 1 + 0.2 * rand(*vec), 0.3 * rand(*vec) if shift else None, 0.5 * rand(*vec) if gate else None
    codes, scale, summed = fl.add_rms_norm_quantize(x, w, r, gate=t, shift=b, blocks=blocks)
    s, y, error = norm_reference(x, w, r, t, b, 1e-6)
    if residual:
        assert summed.dtype == dtype
        terms = r.double().abs() + (s - r.double()).abs()
        assert bool(((summed.double() - s).abs() <= s.abs() * torch.finfo(dtype).eps / 2 + terms * 2.0 ** -23).all())
    else:
        assert summed is None
    if blocks:
        check_quantised(codes, scale, y, error)
    else:
        assert scale.shape == (M, 1)
        want = (y.abs().amax(dim=1, keepdim=True) / 448).clamp_min(1e-12)
        assert bool(((scale.double() - want).abs() <= want * 2.0 ** -23 + error.amax(dim=1, keepdim=True) / 448).all())
        q = y / scale.double()
        assert_nearest_codes(codes, q, 2.0 ** -22 + (error / scale.double()) / q.abs().clamp_min(1e-30))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_in_place_strided_and_one_sample_rows(cuda_device, dtype):
    g = torch.Generator(device=cuda_device).manual_seed(5)
    big = torch.randn(20, 1200, device=cuda_device, generator=g).to(dtype)
    x, r = big[:, 5:645], big[:, 555:1195]
    vecs = torch.randn(2, 3, 640, device=cuda_device, generator=g)  # [samples, (gate, weight, shift), C]
    kwargs = dict(gate=vecs[:, 0], shift=vecs[:, 2])
    want = fl.add_rms_norm_quantize(x.contiguous(), vecs[:, 1].contiguous(), r.contiguous(), gate=vecs[:, 0].contiguous(),
                                    shift=vecs[:, 2].contiguous())
    got = fl.add_rms_norm_quantize(x, vecs[:, 1], r, **kwargs)
    stream = r.clone(memory_format=torch.contiguous_format)
    inplace = fl.add_rms_norm_quantize(x, vecs[:, 1], stream, out=stream, **kwargs)
    assert inplace[2] is stream
    for other in (got, inplace):
        for a, b in zip(want, other):
            assert torch.equal(a.view(torch.uint8), b.contiguous().view(torch.uint8))
    one = fl.add_rms_norm_quantize(x, vecs[0, 1], r, gate=vecs[:1, 0], shift=vecs[0, 2].to(torch.float64))
    two = fl.add_rms_norm_quantize(x, vecs[0, 1], r, gate=vecs[0, 0], shift=vecs[0, 2])
    assert torch.equal(one[0].view(torch.uint8), two[0].view(torch.uint8))


@pytest.mark.gpu
def test_norm_refusals_and_special_values(cuda_device):
    x = torch.randn(6, 256, device=cuda_device)
    w = torch.ones(256, device=cuda_device)
    with pytest.raises(ValueError, match="pass a residual"):
        fl.add_rms_norm_quantize(x, w, gate=w)
    with pytest.raises(ValueError, match="must match x"):
        fl.add_rms_norm_quantize(x, w, x.bfloat16())
    with pytest.raises(ValueError, match="out must be contiguous"):
        fl.add_rms_norm_quantize(x, w, x, out=torch.empty(256, 6, device=cuda_device).t())
    with pytest.raises(ValueError, match="samples"):
        fl.add_rms_norm_quantize(x, w.expand(4, 256), x)
    with pytest.raises(ValueError, match="samples"):
        fl.add_rms_norm_quantize(x, w.expand(2, 256), x, shift=w.expand(3, 256))
    with pytest.raises(ValueError, match="weight must be"):
        fl.add_rms_norm_quantize(x, w[:128])
    with pytest.raises(TypeError, match="float32 and bfloat16"):
        fl.add_rms_norm_quantize(x.half())
    with pytest.raises(RuntimeError, match="same CUDA device"):
        fl.add_rms_norm_quantize(x, w.cpu())
    with pytest.raises(_lib.SparkKernelError, match="at most 16384 columns"):
        fl.add_rms_norm_quantize(torch.randn(2, 16392, device=cuda_device))
    for blocks in (True, False):
        bad = special(x)  # row 0: a NaN, row 5: an infinity, row 3: zeros
        codes, scale, _ = fl.add_rms_norm_quantize(bad, w, blocks=blocks)
        assert bool(codes[0].float().isnan().all()) and bool(scale[0].isnan().all())
        assert bool(codes[5, 128:].float().isnan().all()) and bool(scale[5, -1].isnan())
        assert bool((codes[3].float() == 0).all()) and bool((scale[3] == 1e-12).all())
        assert not bool(codes[[1, 2, 4]].float().isnan().any())
        empty = fl.add_rms_norm_quantize(x[:0], w, x[:0], blocks=blocks)
        assert empty[0].shape == (0, 256) and empty[2].shape == (0, 256)


# ------------------------------------------------------------------------------ GPU: GEMM

def gemm_inputs(M, N, K, device, seed):
    g = torch.Generator(device=device).manual_seed(seed)
    a = (torch.randn(M, K, device=device, generator=g) * 100).clamp(-448, 448).to(E4M3)
    b = (torch.randn(N, K, device=device, generator=g) * 100).clamp(-448, 448).to(E4M3)
    # scales that differ by orders of magnitude from block to block
    a_scale = torch.exp(2 * torch.randn(M, blocks_of(K), device=device, generator=g)) * 1e-3
    b_scale = torch.exp(2 * torch.randn(blocks_of(N), blocks_of(K), device=device, generator=g)) * 1e-3
    return a, a_scale, b, b_scale, g


def gemm_reference(a, a_scale, b, b_scale):
    """(product, bound of its fp32 error) in 64 bits."""
    N, K = b.shape
    da = a.double() * spread(a_scale.double(), K)
    db = b.double() * spread(b_scale.double().repeat_interleave(128, dim=0)[:N], K)
    return da @ db.T, (da.abs() @ db.abs().T) * (128 + blocks_of(K)) * 2.0 ** -23


def assert_gemm(out, want, error):
    assert bool(out.isfinite().all())
    off = (out.double() - want).abs() - want.abs() * torch.finfo(out.dtype).eps / 2 - error
    assert bool((off <= 0).all()), float(off.max())


GEMM_SIZES = [(1, 1, 16), (1, 4096, 4096), (2, 130, 144), (2, 4104, 5376), (3, 1000, 512), (3, 77, 10000), (4, 392, 4112), (4, 5, 16), (8, 512, 128), (9, 1420, 2000), (17, 392, 4112), (24, 1000, 5376),
              (33, 129, 256), (64, 2056, 1024), (65, 640, 640), (100, 4096, 400), (128, 257, 16384), (129, 128, 272),
              (200, 3000, 1040), (256, 256, 128), (259, 5376, 1360), (513, 264, 2064), (1000, 392, 4112), (2100, 4104, 912),
              (1, 28672, 1040), (2, 8200, 4096), (259, 28672, 5376), (2110, 5000, 1040)]


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", GEMM_SIZES)
def test_gemm_matches_its_definition(cuda_device, M, N, K, out_dtype):
    a, a_scale, b, b_scale, _ = gemm_inputs(M, N, K, cuda_device, M + 7 * N + K)
    out = fl.fp8_gemm_blocks(a, a_scale, b, b_scale, out_dtype=out_dtype)
    assert out.shape == (M, N) and out.dtype == out_dtype
    assert_gemm(out, *gemm_reference(a, a_scale, b, b_scale))
    assert ops.read_device_status(cuda_device) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (3, 131, 400), (5, 131, 400), (40, 264, 1040), (130, 520, 2064), (300, 1001, 272),
                                   (2600, 4096, 256)])
def test_gemm_bias_gate_and_residual(cuda_device, M, N, K, out_dtype):
    a, a_scale, b, b_scale, g = gemm_inputs(M, N, K, cuda_device, M + N + K)
    want, error = gemm_reference(a, a_scale, b, b_scale)
    bias = torch.randn(N, device=cuda_device, generator=g) * 10
    gate = torch.randn(N, device=cuda_device, generator=g)
    residual = (torch.randn(M, N, device=cuda_device, generator=g) * 10).to(out_dtype)
    args = (a, a_scale, b, b_scale)
    biased = want + bias.double()
    step = 2.0 ** -23
    assert_gemm(fl.fp8_gemm_blocks(*args, bias, out_dtype=out_dtype), biased, error + (want.abs() + biased.abs()) * step)
    for t in (gate, None):
        f = 1.0 if t is None else t.double()
        full = residual.double() + f * biased
        slack = (torch.as_tensor(f).abs() * (error + (want.abs() + 2 * biased.abs()) * step)) + full.abs() * step
        got = fl.fp8_gemm_blocks(*args, bias, residual=residual, gate=t, out_dtype=out_dtype)
        assert_gemm(got, full, slack)
        into = residual.clone()
        assert fl.fp8_gemm_blocks(*args, bias, residual=into, gate=t, out=into) is into
        assert torch.equal(into, got)


@pytest.mark.gpu
def test_gemm_scale_strides_and_unaligned_operands(cuda_device):
    for M, N, K in ((20, 300, 1040), (400, 300, 1040)):
        a, a_scale, b, b_scale, _ = gemm_inputs(M, N, K, cuda_device, 9)
        want = fl.fp8_gemm_blocks(a, a_scale, b, b_scale)
        wide = torch.empty(M, 3 * a_scale.shape[1], device=cuda_device)
        wide[:, ::3] = a_scale
        for scale in (a_scale.t().contiguous().t(), wide[:, ::3], a_scale.clone()):
            assert torch.equal(fl.fp8_gemm_blocks(a, scale, b, b_scale), want)
        broad = a_scale[:, :1].expand_as(a_scale)
        assert torch.equal(fl.fp8_gemm_blocks(a, broad, b, b_scale), fl.fp8_gemm_blocks(a, broad.contiguous(), b, b_scale))
        padded = torch.zeros(M, K + 16, device=cuda_device).to(E4M3)
        padded[:, 16:] = a
        assert torch.equal(fl.fp8_gemm_blocks(padded[:, 16:], a_scale, b.t().contiguous().t(), b_scale.t().contiguous().t()), want)
        odd = torch.empty(M * K + 1, device=cuda_device, dtype=torch.uint8).view(E4M3)[1:].view(M, K)
        odd.copy_(a)
        with pytest.raises(_lib.SparkKernelError, match="16-byte aligned"):
            fl.fp8_gemm_blocks(odd, a_scale, b, b_scale)


@pytest.mark.gpu
def test_gemm_writes_only_its_output(cuda_device):
    """Rows behind the last one and values past the last column stay as they were."""
    for dtype in (torch.bfloat16, torch.float32):
        for M, N, K in ((1, 4096, 256), (3, 136, 272), (70, 131, 400), (300, 264, 272), (300, 261, 272)):
            a, a_scale, b, b_scale, _ = gemm_inputs(M, N, K, cuda_device, 4)
            buf = torch.full((M + 300, N), 7.0, device=cuda_device, dtype=dtype)
            fl.fp8_gemm_blocks(a, a_scale, b, b_scale, out=buf[:M])
            assert bool((buf[M:] == 7).all())
            assert torch.equal(buf[:M], fl.fp8_gemm_blocks(a, a_scale, b, b_scale, out_dtype=dtype))


@pytest.mark.gpu
def test_gemm_special_values_stay_in_their_rows(cuda_device):
    for M in (6, 300):
        a, a_scale, b, b_scale, _ = gemm_inputs(M, 260, 400, cuda_device, 8)
        clean = fl.fp8_gemm_blocks(a, a_scale, b, b_scale)
        a_bad, s_bad = a.clone(), a_scale.clone()
        a_bad.view(torch.uint8)[2, 130] = 0x7F  # NaN
        s_bad[4, 1] = float("inf")
        out = fl.fp8_gemm_blocks(a_bad, s_bad, b, b_scale)
        assert bool(out[2].isnan().all()) and not bool(out[4].isfinite().any())
        keep = [m for m in range(M) if m not in (2, 4)]
        assert torch.equal(out[keep], clean[keep])
        zero = torch.zeros_like(a_scale)
        assert bool((fl.fp8_gemm_blocks(a, zero, b, b_scale) == 0).all())


@pytest.mark.gpu
def test_gemm_refusals_and_empty(cuda_device):
    a, a_scale, b, b_scale, _ = gemm_inputs(4, 200, 256, cuda_device, 1)
    bad = [
        (lambda: fl.fp8_gemm_blocks(a.float(), a_scale, b, b_scale), TypeError, "float8_e4m3fn"),
        (lambda: fl.fp8_gemm_blocks(a, a_scale, b[:, :128], b_scale), ValueError, "share K"),
        (lambda: fl.fp8_gemm_blocks(a, a_scale[:, :1], b, b_scale), ValueError, "a_scale must be"),
        (lambda: fl.fp8_gemm_blocks(a, a_scale.double(), b, b_scale), TypeError, "a_scale must be float32"),
        (lambda: fl.fp8_gemm_blocks(a, a_scale, b, b_scale[:1]), ValueError, "b_scale must be"),
        (lambda: fl.fp8_gemm_blocks(a, a_scale, b, b_scale, a_scale[0]), ValueError, "bias needs 200"),
        (lambda: fl.fp8_gemm_blocks(a, a_scale, b, b_scale, gate=a_scale[0]), ValueError, "pass a residual"),
        (lambda: fl.fp8_gemm_blocks(a, a_scale, b, b_scale, residual=torch.ones(4, 200, device=cuda_device)), ValueError,
         "residual must be"),
        (lambda: fl.fp8_gemm_blocks(a, a_scale, b, b_scale, out_dtype=torch.float16), TypeError, "float32 and bfloat16"),
        (lambda: fl.fp8_gemm_blocks(a, a_scale, b, b_scale, out=torch.empty(200, 4, device=cuda_device).t()), ValueError,
         "out must be contiguous"),
        (lambda: fl.fp8_gemm_blocks(a, a_scale.cpu(), b, b_scale), RuntimeError, "same CUDA device"),
        (lambda: fl.fp8_gemm_blocks(a[:, :250], a_scale, b[:, :250], b_scale), _lib.SparkKernelError, "multiple of 16"),
    ]
    for call, error, match in bad:
        with pytest.raises(error, match=match):
            call()
    assert fl.fp8_gemm_blocks(a[:0], a_scale[:0], b, b_scale).shape == (0, 200)
    assert fl.fp8_gemm_blocks(a, a_scale, b[:0], b_scale[:0]).shape == (4, 0)


# ------------------------------------------------------------------------------ GPU: together

@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 7, 60, 300])
def test_chain_on_another_stream_and_in_a_graph(cuda_device, M):
    """norm -> up projection -> SwiGLU -> down projection with its residual, as a block runs them:
    on a side stream and as a replayed graph, bit for bit as eagerly."""
    g = torch.Generator(device=cuda_device).manual_seed(M)
    C, inner = 512, 1040
    up = fl.quantize_weight_blocks(torch.randn(2 * inner, C, device=cuda_device, generator=g) * 0.04)
    down = fl.quantize_weight_blocks(torch.randn(C, inner, device=cuda_device, generator=g) * 0.04)
    weight = 1 + 0.1 * torch.randn(C, device=cuda_device, generator=g)
    delta = torch.randn(M, C, device=cuda_device, generator=g).to(torch.bfloat16)
    stream_in = torch.randn(M, C, device=cuda_device, generator=g).to(torch.bfloat16)

    def block():
        codes, scale, s = fl.add_rms_norm_quantize(delta, weight, stream_in)
        h = fl.fp8_gemm_blocks(codes, scale, *up)
        act, act_scale = fl.swiglu_quantize_blocks(h)
        return fl.fp8_gemm_blocks(act, act_scale, *down, residual=s)

    eager = block()
    # the same block in 64 bits from the same weights: e4m3 activations keep three bits
    n = delta.double() + stream_in.double()
    y = n * torch.rsqrt(n.square().mean(1, keepdim=True) + 1e-6) * weight.double()
    w_up = up[0].double() * spread(up[1].double().repeat_interleave(128, 0)[:2 * inner], C)
    w_down = down[0].double() * spread(down[1].double().repeat_interleave(128, 0)[:C], inner)
    h = y @ w_up.T
    act = h[:, :inner] * h[:, inner:] * torch.sigmoid(h[:, inner:])
    want = n + act @ w_down.T
    assert F.cosine_similarity((eager.double() - n).flatten(), (want - n).flatten(), dim=0) > 0.995
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        other = block()
    torch.cuda.current_stream(cuda_device).wait_stream(side)
    assert torch.equal(other, eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = block()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, eager)
    delta.mul_(0.5)
    graph.replay()
    again = block()
    torch.cuda.synchronize()
    assert torch.equal(captured, again) and not torch.equal(again, eager)
    del graph


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_block_linear_close_to_the_linear(cuda_device, dtype):
    torch.manual_seed(25)
    linear = nn.Linear(1040, 2056, bias=True, device=cuda_device, dtype=dtype)
    with torch.no_grad():
        linear.weight[:, 5] *= 40  # one outlier channel
    x = torch.randn(3, 43, 1040, device=cuda_device, dtype=dtype)
    with torch.no_grad():
        want, got = linear(x), fl.Fp8BlockLinear(linear)(x)
    assert got.shape == want.shape and got.dtype == dtype
    # Two roundings to e4m3, each at most 2^-4 of a value.  Over a binade's values the root mean
    # square of one is about 2^-4 / sqrt(6), and independent errors of a sum's terms leave the
    # sum's relative error there: sqrt(2) 2^-4 / sqrt(6) < 2^-4.  (No smaller than per-channel
    # scales': e4m3 is a floating type, so a scale matters only to values near its subnormals.)
    assert float((got.float() - want.float()).norm() / want.float().norm()) <= 2.0 ** -4


@pytest.mark.gpu
def test_install_with_block_scales(cuda_device):
    from test_fp8_linear import FeedForward
    from test_gpu_plugin import TinyAttention

    torch.manual_seed(28)
    attn = TinyAttention(hidden=128, heads=1).to(cuda_device, torch.bfloat16).eval()
    block = nn.Module()
    block.attn = attn
    block.ff = FeedForward(dim=128, inner=272).to(cuda_device, torch.bfloat16).eval()
    model = nn.Module()
    model.transformer_blocks = nn.ModuleList([block])
    x = torch.randn(1, 259, 128, device=cuda_device, dtype=torch.bfloat16)
    with torch.no_grad():
        q = attn.to_q(x)
        ff = block.ff(x)
        assert fl.install_fp8(model, min_width=8, skip_end_blocks=0, scales="block") == 5
        assert type(attn.get_processor()) is fl.Fp8AttnProcessor and type(block.ff) is fl.Fp8SwiGLUFeedForward
        shared = fl.forward_qkv_shared(attn, x)
        assert torch.equal(shared[0], attn.to_q(x))
        assert F.cosine_similarity(shared[0].flatten().float(), q.flatten().float(), dim=0) > 0.998
        assert F.cosine_similarity(block.ff(x).flatten().float(), ff.flatten().float(), dim=0) > 0.995
        assert attn(x).isfinite().all()
        attn.to_k = nn.Linear(128, 128, bias=False, device=cuda_device, dtype=torch.bfloat16)
        assert fl.forward_qkv_shared(attn, x) is None
        attn.to_k = fl.Fp8Linear(attn.to_k)
        assert fl.forward_qkv_shared(attn, x) is None  # another granularity


def test_stack_rejects_unknown_linear_scales():
    from spark_h3_b200.dit import DiTConfig, DiTStack

    cfg = DiTConfig(hidden=256, heads=2, ffn=512, blocks=1)
    with pytest.raises(ValueError, match="linear_scales"):
        DiTStack(cfg, (1, 4, 8), device="cpu", linear_scales="tensor")
    with pytest.raises(ValueError, match="peer_exchange"):
        DiTStack(cfg, (1, 4, 8), device="cpu", linear_scales="block", peer_exchange=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dense", [True, False])
def test_stack_step_with_block_scales(cuda_device, dense):
    """The DiT stack with block-scaled linears against the fp32 restatement of its block, to the
    bounds of the per-channel stack's own test."""
    from spark_h3_b200.attention import spark_attention_bthd
    from spark_h3_b200.dit import DiTConfig, DiTStack, reference_block_math

    cfg = DiTConfig(hidden=256, heads=2, ffn=512, blocks=2)
    stack = DiTStack(cfg, (2, 16, 32), device=cuda_device, seed=3, spark_mode="reweight_only", topk_ratio=0.2,
                     linear_scales="block")
    g = torch.Generator(device=cuda_device).manual_seed(5)
    x0 = torch.randn(stack.local, cfg.hidden, device=cuda_device, generator=g).to(torch.bfloat16)
    x = stack.step(x0.clone(), 500.0, dense=dense)

    def attention(q, k, v):
        if dense:
            o = F.scaled_dot_product_attention(q.float().transpose(1, 2), k.float().transpose(1, 2),
                                               v.float().transpose(1, 2))
            return o.transpose(1, 2).to(torch.bfloat16)
        return spark_attention_bthd(stack.controller, q.contiguous(), k.contiguous(), v.contiguous(), stack.layout, 0)

    ref = x0
    for blk, mod in zip(stack.blocks, stack.modulation(500.0)):
        ref = reference_block_math(ref, blk, mod, cfg, stack.coords, stack.inv_freq, stack.axis, attention, "block")
    diff = (x.float() - ref.float()).abs().max().item()
    cos = F.cosine_similarity(x.float().flatten(), ref.float().flatten(), dim=0).item()
    assert torch.isfinite(x).all()
    assert cos > 0.999 and diff <= 0.05 * ref.float().abs().max().item(), (cos, diff)


@pytest.mark.gpu
def test_attention_segments_quantise_in_row_order(cuda_device):
    """Codes and scales of two ranks' head segments, put in row order, are those of the rows."""
    M, hp = 50, 2
    seg = torch.randn(2, M, hp * 128, device=cuda_device).to(torch.bfloat16)
    rows = seg.transpose(0, 1).reshape(M, -1)
    codes, scale = fl.quantize_blocks(seg.view(2 * M, -1))
    got = tuple(t.view(2, M, -1).transpose(0, 1).reshape(M, -1) for t in (codes, scale))
    want = fl.quantize_blocks(rows)
    assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])


# ------------------------------------------------------------------------------ GPU: far offsets, neighbours, streams

@pytest.mark.gpu
def test_offsets_past_32_bits(cuda_device):
    """Rows that start past 2^31 elements: the last rows of a large call are those of a small one."""
    M, K, tail = 140_000, 16_384, 5  # 2.3e9 elements
    assert M * K > 2 ** 31
    x = torch.zeros(M, K, device=cuda_device, dtype=torch.bfloat16)
    x[-tail:] = torch.randn(tail, K, device=cuda_device).to(torch.bfloat16)
    weight = torch.randn(K, device=cuda_device)
    for call in (fl.quantize_blocks, fl.swiglu_quantize_blocks, lambda t: fl.add_rms_norm_quantize(t, weight)[:2]):
        got, want = call(x), call(x[-tail:])
        for a, b in zip(got, want):
            assert torch.equal(a[-tail:].view(torch.uint8), b.view(torch.uint8))
        del got
    summed = fl.add_rms_norm_quantize(x, weight, x, out=x)[2]
    assert summed is x and bool((x[:-tail] == 0).all())
    del x, summed
    for N, dtype in ((16_600, torch.bfloat16), (16_601, torch.bfloat16)):  # TMA stores, row by row stores
        a, a_scale, b, b_scale, _ = gemm_inputs(131_000, N, 16, cuda_device, 2)
        assert a.shape[0] * N > 2 ** 31
        out = fl.fp8_gemm_blocks(a, a_scale, b, b_scale, out_dtype=dtype)
        assert torch.equal(out[-300:], fl.fp8_gemm_blocks(a[-300:], a_scale[-300:], b, b_scale, out_dtype=dtype))
        del out


@pytest.mark.gpu
@pytest.mark.parametrize("K", [256, 264, 131])
def test_kernels_leave_the_memory_around_their_outputs(cuda_device, K):
    M, pad = 9, 512
    x = torch.randn(M, K, device=cuda_device)
    nb = blocks_of(K)
    stream = torch.cuda.current_stream(cuda_device).cuda_stream

    def guarded(n, dtype):
        buf = torch.full((n + 2 * pad,), 77, device=cuda_device, dtype=dtype)
        return buf, buf[pad:].data_ptr()

    codes, codes_ptr = guarded(M * K, torch.uint8)
    scale, scale_ptr = guarded(M * nb, torch.float32)
    summed, summed_ptr = guarded(M * K, torch.float32)
    _lib.call("sb_fp8_quantize_blocks", x.data_ptr(), K, _lib.F32, M, K, codes_ptr, scale_ptr, stream)
    _lib.call("sb_fp8_add_rms_norm_quantize", x.data_ptr(), K, x.data_ptr(), K, None, 0, None, 0, None, 0, _lib.F32, M, K,
              M, 1e-6, 1, summed_ptr, codes_ptr, scale_ptr, stream)
    for buf, n in ((codes, M * K), (scale, M * nb), (summed, M * K)):
        assert bool((buf[:pad] == 77).all()) and bool((buf[pad + n:] == 77).all())
    want = fl.add_rms_norm_quantize(x, None, x)
    assert torch.equal(codes[pad:pad + M * K].view(M, K), want[0].view(torch.uint8))
    assert torch.equal(summed[pad:pad + M * K].view(M, K), want[2])


@pytest.mark.gpu
def test_calls_on_two_streams_at_once(cuda_device):
    """Split, streamed and paired GEMMs of different shapes overlap on two streams without touching
    each other's results (there is no shared workspace)."""
    shapes = [(2, 4096, 4096), (40, 1024, 4096), (300, 2056, 1040), (16, 4104, 5376)]
    cases = []
    for i, s in enumerate(shapes):
        args = gemm_inputs(*s, cuda_device, 20 + i)[:4]
        cases.append((args, fl.fp8_gemm_blocks(*args)))
    streams = [torch.cuda.Stream(cuda_device) for _ in range(2)]
    outs = []
    torch.cuda.synchronize()
    for round_ in range(12):
        for i, stream in enumerate(streams):
            args, want = cases[(round_ + 2 * i) % len(cases)]
            with torch.cuda.stream(stream):
                outs.append((fl.fp8_gemm_blocks(*args), want))
    torch.cuda.synchronize()
    assert all(torch.equal(got, want) for got, want in outs)
    assert ops.read_device_status(cuda_device) == 0


@pytest.mark.gpu
def test_results_do_not_change_from_call_to_call(cuda_device):
    for s in ((1, 4096, 4096), (24, 14336, 1040), (64, 512, 16384), (2600, 4096, 1040)):
        args = gemm_inputs(*s, cuda_device, 3)[:4]
        first = fl.fp8_gemm_blocks(*args, out_dtype=torch.float32)
        for _ in range(5):
            assert torch.equal(fl.fp8_gemm_blocks(*args, out_dtype=torch.float32), first)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(300, 1001, 272), (2600, 4099, 400), (520, 131, 1040)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gemm_odd_columns_with_residual_in_place(cuda_device, M, N, K, dtype):
    """Rows that are no whole 16-byte vectors go through shared memory in both directions."""
    a, a_scale, b, b_scale, g = gemm_inputs(M, N, K, cuda_device, M)
    want, error = gemm_reference(a, a_scale, b, b_scale)
    residual = (torch.randn(M, N, device=cuda_device, generator=g) * 10).to(dtype)
    full = residual.double() + want
    out = fl.fp8_gemm_blocks(a, a_scale, b, b_scale, residual=residual, out=residual)
    assert out is residual
    assert_gemm(out, full, error + (want.abs() + full.abs()) * 2.0 ** -23)


def test_block_scales_leave_unfit_linears():
    """in_features that is no multiple of 16 (the GEMM's row pitch): the Linear stays."""
    model = nn.Module()
    model.transformer_blocks = nn.ModuleList([nn.Sequential(nn.Linear(24, 32), nn.Linear(32, 24))])
    assert fl.convert_linear_to_fp8(model, min_width=8, scales="block") == 1
    assert type(model.transformer_blocks[0][0]) is nn.Linear
    assert type(model.transformer_blocks[0][1]) is fl.Fp8BlockLinear


@pytest.mark.gpu
def test_outputs_that_overlap_an_input_are_refused(cuda_device):
    buf = torch.randn(9, 256, device=cuda_device).to(torch.bfloat16)
    with pytest.raises(ValueError, match="overlaps residual"):
        fl.add_rms_norm_quantize(torch.randn(8, 256, device=cuda_device).to(torch.bfloat16), None, buf[:8], out=buf[1:])
    wide = torch.randn(8, 512, device=cuda_device).to(torch.bfloat16)
    with pytest.raises(ValueError, match="overlaps x"):  # the same address, another layout
        fl.add_rms_norm_quantize(wide[:, :256], None, buf[:8], out=wide.view(-1)[:8 * 256].view(8, 256))
    a, a_scale, b, b_scale, _ = gemm_inputs(8, 256, 256, cuda_device, 1)
    with pytest.raises(ValueError, match="overlaps residual"):
        fl.fp8_gemm_blocks(a, a_scale, b, b_scale, residual=buf[:8], out=buf[1:])
    a, a_scale, b, b_scale, _ = gemm_inputs(8, 128, 256, cuda_device, 1)
    with pytest.raises(ValueError, match="overlaps a_fp8"):
        fl.fp8_gemm_blocks(a, a_scale, b, b_scale, out=a.view(torch.bfloat16))  # [8, 128]


@pytest.mark.gpu
def test_processor_projects_one_by_one_where_granularities_differ(cuda_device):
    from test_gpu_plugin import TinyAttention

    torch.manual_seed(4)
    attn = TinyAttention(hidden=128, heads=1).to(cuda_device, torch.bfloat16).eval()
    x = torch.randn(1, 70, 128, device=cuda_device, dtype=torch.bfloat16)
    processor = fl.Fp8AttnProcessor()
    with torch.no_grad():
        attn.to_q, attn.to_v = fl.Fp8BlockLinear(attn.to_q), fl.Fp8BlockLinear(attn.to_v)
        mixed = processor(attn, x)
        attn.to_k = fl.Fp8BlockLinear(attn.to_k)
        shared = processor(attn, x)
    assert mixed.isfinite().all() and F.cosine_similarity(mixed.flatten().float(), shared.flatten().float(), dim=0) > 0.99
    empty = fl.Fp8BlockLinear(nn.Linear(64, 32, device=cuda_device, dtype=torch.bfloat16))
    assert empty(x.new_empty(0, 64)).shape == (0, 32)
