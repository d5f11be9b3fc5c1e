"""GPU: fp32 results of the grouped W8A8 products against their definition in 64 bits."""
import pytest
import torch

import w8a8_reference as R
from mini_qwen_b200.kernels import w8a8_grouped_swiglu, w8a8_grouped_swiglu_gather

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("N", [16, 144, 17])              # CTA pairs, and the small tiles that take any width
@pytest.mark.parametrize("gather", [False, True])
def test_swiglu_keeps_fp32_over_the_whole_range(N, gather):
    """Whole numbers and powers of two: g = q 2^j and u are exact, so the result is off by its own arithmetic alone.  The
    exponential is off by 2^-22 relative, the reciprocal by 2^-23, the correction, the sum and the three products by half a unit
    each (5 * 2^-24): below 12 * 2^-24.  Where the exponential is below 2^-126 it has the step of the smallest numbers, 2^-149,
    twice (itself and its correction), which |g u| multiplies."""
    K = 32
    q = torch.arange(-127, 128, device=DEV)
    x = torch.zeros(255, K, dtype=torch.int8, device=DEV)
    x[:, 0], x[:, 1] = q.to(torch.int8), 96
    w = torch.zeros(1, 2 * N, K, dtype=torch.int8, device=DEV)
    w[0, :N, 0], w[0, N:, 1] = 1, 1
    scales = torch.ones(1, 2 * N, device=DEV)
    scales[0, :N] = 2.0 ** -(torch.arange(N, device=DEV) % 6).float()
    sx = torch.ones(255, device=DEV)
    off = torch.tensor([0, 255], dtype=torch.int32, device=DEV)
    if gather:
        perm = torch.arange(254, -1, -1, dtype=torch.int32, device=DEV)
        out = w8a8_grouped_swiglu_gather(x, perm, 1, w, scales, off, x_scale=sx, out_dtype=torch.float32).flip(0)
    else:
        out = w8a8_grouped_swiglu(x, w, scales, off, x_scale=sx, out_dtype=torch.float32)
    g, u = R.product(x.double(), sx.double(), w[0], scales[0].double()).chunk(2, dim=1)
    ref = g * torch.sigmoid(g) * u
    bound = ref.abs() * 12 * 2.0 ** -24 + (g * u).abs() * 2.0 ** -148
    worst = ((out.double() - ref).abs() - bound).max()
    assert float(worst) <= 0, f"off by {float(((out.double() - ref).abs() / ref.abs().clamp_min(1e-300)).max())} of the value"
