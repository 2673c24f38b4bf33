"""Block-scaled e4m3 operators where they meet the edges of their arithmetic and of their arguments:
SwiGLU of values whose product overflows, GELU's negative tail, outputs that are inputs,
linears of different kinds side by side, one and two rows of A on both sides of their kernels' border, and the registers that
the kernels' launches count on."""
from __future__ import annotations

import re
import subprocess

import pytest
import torch
import torch.nn as nn

from spark_h3_b200 import _build, fp8_linear as fl, ops
from spark_h3_b200.processor import _H3SparseProcessor
from test_fp8_blocks import assert_gemm, check_quantised, gemm_inputs, gemm_reference


# ------------------------------------------------------------------------------ SwiGLU

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [128, 130, 131])
def test_swiglu_of_values_whose_product_overflows(cuda_device, dtype, K):
    """a * silu(g) is finite (or vanishes) where a * g alone is past fp32's largest value."""
    pairs = [(3e38, -10.0), (-3e38, -30.0), (3e38, 1.2), (-2.5e38, -1.5), (3e38, -200.0), (-1e30, -1e9), (1e38, -5.5)]
    h = torch.zeros(len(pairs), 2 * K, device=cuda_device)
    for row, (a, g) in enumerate(pairs):
        h[row, K - 1], h[row, 2 * K - 1] = a, g
        if abs(a) < 1e36:
            h[row, 0], h[row, K] = 1.0, 1.0  # beside an ordinary value
    h = h.to(dtype)
    a, g = h.double().chunk(2, dim=1)
    y = a * (g * torch.sigmoid(g))
    # exp's argument is off by |g| 2^-23, its value by 2^-22, four more operations by 2^-23 each
    check_quantised(*fl.swiglu_quantize_blocks(h), y, y.abs() * (g.abs() * 2.0 ** -23 + 2.0 ** -20))


# ------------------------------------------------------------------------------ GELU

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K", [(64, 129), (33, 131), (40, 258), (9, 4096)])
@pytest.mark.parametrize("low,high", [(-6.0, -1.0), (-4.0, -3.0), (-9.0, 9.0)])
def test_gelu_is_exact_relative_to_its_value(cuda_device, dtype, M, K, low, high):
    """A group may hold nothing but GELU's negative tail (a short last group often does): its scale
    and codes need the tail's relative accuracy."""
    g = torch.Generator(device=cuda_device).manual_seed(K)
    x = (torch.rand(M, K, device=cuda_device, generator=g) * (high - low) + low).to(dtype)
    y = x.double() * torch.special.ndtr(x.double())
    # Phi(-|x|) e^(x^2 / 2) as a polynomial in t: its fit 3e-7, t (off by 2^-24 + 2^-23) three times
    # that, seven steps of Horner's rule 1.5e-6, two products and ex2 (2^-22): 2.8e-6 < 2^-18.  The
    # exponent x^2 / 2 is off by two roundings and its constant's, 2.5 x 2^-24 of itself.
    error = y.abs() * (2.0 ** -18 + x.double().square() * 1.25 * 2.0 ** -24)
    check_quantised(*fl.gelu_quantize_blocks(x), y, error)


# ------------------------------------------------------------------------------ the same call again

@pytest.mark.gpu
@pytest.mark.parametrize("act", [fl.quantize_blocks, fl.swiglu_quantize_blocks, fl.gelu_quantize_blocks])
def test_quantisers_give_the_same_bits_again(cuda_device, act):
    """Whichever stream, address and number of rows beside them: a row's codes and scales are its own."""
    x = torch.randn(259, 2 * 1432, device=cuda_device).to(torch.bfloat16)
    codes, scale = act(x)
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        others = [act(x), act(x.clone()), act(x[:3]), act(torch.nn.functional.pad(x, (1, 0))[:, 1:])]
    torch.cuda.current_stream(cuda_device).wait_stream(side)
    for got in others:
        rows = got[0].shape[0]
        assert torch.equal(got[0].view(torch.uint8), codes[:rows].view(torch.uint8)) and torch.equal(got[1], scale[:rows])


# ------------------------------------------------------------------------------ outputs that are inputs

@pytest.mark.gpu
def test_out_is_no_operand_that_others_still_read(cuda_device):
    x = torch.randn(4, 256, device=cuda_device)
    for name in ("weight", "shift", "gate"):
        vec = torch.randn(4, 256, device=cuda_device)  # one sample per row: out's shape and type
        kept = vec.clone()
        with pytest.raises(ValueError, match=f"overlaps {name}"):
            fl.add_rms_norm_quantize(x, residual=x, out=vec, **{name: vec})
        assert torch.equal(vec, kept)
    a = torch.ones(4, 512, device=cuda_device).to(fl.FP8_DTYPE)
    b = torch.ones(4, 512, device=cuda_device).to(fl.FP8_DTYPE)
    a_scale, b_scale = torch.rand(4, 4, device=cuda_device), torch.rand(1, 4, device=cuda_device)
    with pytest.raises(ValueError, match="overlaps a_scale"):
        fl.fp8_gemm_blocks(a, a_scale, b, b_scale, out=a_scale)
    with pytest.raises(ValueError, match="overlaps b_scale"):
        fl.fp8_gemm_blocks(a[:1], a_scale[:1], b, b_scale, out=b_scale)
    row = torch.rand(1, 4, device=cuda_device)
    with pytest.raises(ValueError, match="overlaps bias"):
        fl.fp8_gemm_blocks(a[:1], a_scale[:1], b, b_scale, row, out=row)
    with pytest.raises(ValueError, match="overlaps gate"):
        fl.fp8_gemm_blocks(a[:1], a_scale[:1], b, b_scale, residual=torch.rand(1, 4, device=cuda_device), gate=row, out=row)


def test_only_inputs_read_in_place_may_be_the_output():
    out = torch.zeros(4, 8)
    fl._refuse_overlap(out, dict(x=out, residual=None), weight=torch.zeros(8))
    fl._refuse_overlap(out, dict(x=torch.zeros(4, 8)))
    with pytest.raises(ValueError, match="overlaps weight$"):
        fl._refuse_overlap(out, dict(x=out), weight=out)
    with pytest.raises(ValueError, match="overlaps shift$"):
        fl._refuse_overlap(out, dict(x=out), shift=out[3])
    with pytest.raises(ValueError, match="overlaps x without being it"):
        fl._refuse_overlap(out, dict(x=out.as_strided((4, 8), (1, 4))))


# ------------------------------------------------------------------------------ mixed projections

class Attention(nn.Module):
    """What the sparse processor's projections read of an attention module."""

    def __init__(self, hidden, heads):
        super().__init__()
        self.heads, self.fused_projections = heads, False
        self.to_q, self.to_k, self.to_v = (nn.Linear(hidden, hidden, bias=False) for _ in range(3))
        self.norm_q = self.norm_k = nn.Identity()


class HostFp8Linear(fl.Fp8Linear):
    """An Fp8Linear whose product is taken on the CPU from its codes and scales."""

    def forward(self, x):
        return x @ (self.weight_fp8.float() * self.weight_scale.reshape(-1, 1)).T


@pytest.mark.parametrize("which", [("to_q",), ("to_q", "to_v"), ("to_k",), ()])
def test_sparse_processor_projects_fp8_beside_plain_linears(which):
    torch.manual_seed(6)
    attn = Attention(32, 2)
    for name in which:
        setattr(attn, name, HostFp8Linear(getattr(attn, name)))
    x = torch.randn(1, 7, 32)
    with torch.no_grad():
        got = _H3SparseProcessor._project(attn, x, None)
        for t, linear in zip(got, (attn.to_q, attn.to_k, attn.to_v)):
            assert torch.equal(t, linear(x).unflatten(-1, (2, 16)))


@pytest.mark.gpu
def test_sparse_processor_projects_mixed_granularities(cuda_device):
    torch.manual_seed(7)
    attn = Attention(256, 2).to(cuda_device, torch.bfloat16)
    plain = [m for m in (attn.to_q, attn.to_k, attn.to_v)]
    attn.to_q, attn.to_k = fl.Fp8Linear(attn.to_q), fl.Fp8BlockLinear(attn.to_k)
    x = torch.randn(1, 70, 256, device=cuda_device, dtype=torch.bfloat16)
    with torch.no_grad():
        got = _H3SparseProcessor._project(attn, x, None)
        for t, linear, before in zip(got, (attn.to_q, attn.to_k, attn.to_v), plain):
            assert torch.equal(t, linear(x).unflatten(-1, (2, 128)))
            # two roundings to e4m3 (2^-4 of a value at most): root mean square below 2^-4 together
            want = before(x).float().flatten()
            assert float((t.float().flatten() - want).norm() / want.norm()) <= 2.0 ** -4


# ------------------------------------------------------------------------------ one and two rows

@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (1, 5376, 4096), (1, 4096, 4112), (1, 23000, 1024), (1, 512, 16384),
                                   (2, 2048, 4096), (2, 2368, 4096), (2, 2369, 4096), (2, 4096, 4096), (2, 8192, 2048),
                                   (2, 1536, 16384), (2, 7, 4112), (1, 1, 8208), (2, 40000, 16), (1, 40000, 16)])
def test_one_and_two_rows_at_the_border_of_their_kernels(cuda_device, M, N, K):
    a, a_scale, b, b_scale, g = gemm_inputs(M, N, K, cuda_device, N + K)
    want, error = gemm_reference(a, a_scale, b, b_scale)
    assert_gemm(fl.fp8_gemm_blocks(a, a_scale, b, b_scale, out_dtype=torch.float32), want, error)
    residual = torch.randn(M, N, device=cuda_device, generator=g).to(torch.bfloat16)
    full = residual.double() + want
    out = fl.fp8_gemm_blocks(a, a_scale, b, b_scale, residual=residual, out=residual)
    assert_gemm(out, full, error + full.abs() * 2.0 ** -23)
    assert ops.read_device_status(cuda_device) == 0


# ------------------------------------------------------------------------------ registers

def test_kernels_have_the_registers_that_their_launches_count_on(tmp_path):
    """The pair kernel refuses to run with another count than the one its warps redistribute, and the
    choice of the streaming kernel counts four CTAs per SM for one row, two for two."""
    source = _build.CSRC_DIR / "fp8_gemm_blocks.cu"
    log = subprocess.run([_build._nvcc(), *_build.NVCC_FLAGS, "-I", str(_build.INCLUDE_DIR), "-Xptxas", "-v", "-c",
                          str(source), "-o", str(tmp_path / "out.o")], capture_output=True, text=True, check=True).stderr
    used = {name: int(count) for name, count in
            re.findall(r"entry function '([^']+)'.*?Used (\d+) registers", log, flags=re.S)}
    launch = int(re.search(r"kLaunchRegs = (\d+)", source.read_text()).group(1))
    pair = [n for name, n in used.items() if "pair_kernel" in name]
    assert len(pair) == 2 and set(pair) == {launch}
    for rows, resident in ((1, 4), (2, 2)):
        stream = [n for name, n in used.items() if "stream_kernel" in name and f"Li{rows}E" in name]
        assert len(stream) == 2
        for n in stream:  # registers come in eights per thread, 65,536 to an SM
            assert 65536 // (-(-n // 8) * 8 * 256) == resident


# ------------------------------------------------------------------------------ infinities and NaN

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_activations_of_infinities_and_nan(cuda_device, dtype):
    """A NaN takes its group of 128, an infinity its group's finite values; the other groups stay."""
    x = torch.randn(6, 300, device=cuda_device).to(dtype)
    x[0, 130], x[1, 5], x[2, 299] = float("nan"), float("inf"), float("-inf")
    x[3, 0], x[4, 0] = 3e38, -3e38
    codes, scale = fl.gelu_quantize_blocks(x)
    clean = fl.gelu_quantize_blocks(x.nan_to_num(1.0, 1.0, 1.0))
    assert bool(codes[0, 128:256].float().isnan().all()) and bool(scale[0, 1].isnan())
    assert bool(scale[1, 0].isinf()) and bool(codes[1, 5].float().isnan())
    assert bool((codes[1, :128].float().nan_to_num(0.0) == 0).all())
    assert bool(codes[2, 256:].float().isnan().all())  # -inf * Phi(-inf) is no number, as in torch
    assert bool(scale[3, 0] > 6e35) and bool((codes[4, 0].float() == 0))
    hit = torch.zeros(6, 3, dtype=torch.bool, device=cuda_device)
    hit[0, 1] = hit[1, 0] = hit[2, 2] = True
    assert torch.equal(scale[~hit], clean[1][~hit])
    h = torch.randn(4, 600, device=cuda_device).to(dtype)
    h[0, 3], h[1, 300 + 140], h[2, 7], h[2, 300 + 7] = float("nan"), float("nan"), float("inf"), 1.0
    h[3, 9], h[3, 300 + 9] = 1.0, float("inf")
    codes, scale = fl.swiglu_quantize_blocks(h)
    assert bool(codes[0, :128].float().isnan().all()) and bool(codes[1, 128:256].float().isnan().all())
    assert not bool(codes[0, 128:].float().isnan().any()) and not bool(codes[1, :128].float().isnan().any())
    for row, column in ((2, 7), (3, 9)):
        assert bool(scale[row, 0].isinf()) and bool(codes[row, column].float().isnan())
        assert bool((codes[row, :128].float().nan_to_num(0.0) == 0).all()) and bool(scale[row, 1:].isfinite().all())
