"""Block-scaled e4m3 operators where they meet the edges of their arithmetic and of their arguments:
SwiGLU of values whose product overflows."""
from __future__ import annotations

import pytest
import torch

from spark_h3_b200 import fp8_linear as fl
from test_fp8_blocks import check_quantised


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
