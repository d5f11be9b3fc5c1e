"""GPU: the grouped W8A8 products against their definition in 64 bits: fp32 results, numbers of 128-k blocks that are odd, many
groups."""
import pytest
import torch

import w8a8_reference as R
from mini_qwen_b200.kernels import w8a8_grouped_gemm, w8a8_grouped_swiglu, w8a8_grouped_swiglu_gather

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


def check_experts(counts, K, N, dtype, period=None):
    """All three grouped products of groups of these rows, group g on expert g % period."""
    S, E = sum(counts), period or len(counts)
    g = torch.Generator(device=DEV).manual_seed(S + K + N)
    x = torch.randn(S, K, generator=g, device=DEV).to(dtype)
    w = torch.randint(-128, 128, (E, N, K), generator=g, device=DEV, dtype=torch.int8)
    s = torch.rand(E, N, generator=g, device=DEV) * 0.01 + 1e-4
    off = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = w8a8_grouped_gemm(x, w, s, off, status=status)
    h = w8a8_grouped_swiglu(x, w, s * 0.05, off, status=status)
    perm = torch.randperm(S, generator=g, device=DEV).to(torch.int32)
    back = torch.empty_like(x)
    back[perm.long()] = x
    gathered = w8a8_grouped_swiglu_gather(back, perm, 1, w, s * 0.05, off, status=status)
    assert status.item() == 0 and out.dtype == h.dtype == dtype
    q, sx = R.quantize(x)
    lo = 0
    for i, n in enumerate(counts):
        rows, e = slice(lo, lo + n), i % E
        R.assert_close(out[rows], R.product(q[rows], sx[rows], w[e], s[e]))
        ref, size = R.swiglu(q[rows], sx[rows], w[e], s[e] * 0.05)
        R.assert_close(h[rows], ref, R.swiglu_extra(size))
        R.assert_close(gathered[rows], ref, R.swiglu_extra(size))
        lo += n


COUNTS = [[1], [1, 0, 31, 32, 33], [128, 129, 0, 256, 257, 1], [512, 513, 545, 2, 1025], [20] * 20 + [1100] + [300, 20] + [7, 0, 31] * 16]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K,N", [(128, 256), (272, 128), (640, 272), (256, 128), (100, 50)])
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{max(c)}")
def test_experts(counts, K, N, dtype):
    """1, 3 and 5 blocks of 128 k: where a stage takes two, the second half of the last lies past K and has to count all the
    same."""
    check_experts(counts, K, N, dtype)


@pytest.mark.parametrize("groups,period", [(300, 300), (1020, 60), (1100, 1100), (1100, 100)])
def test_many_groups(groups, period):
    """Over 256 groups are not put in order of size, over 1024 go to the small tiles; some are empty, one is large."""
    counts = [(7 * i) % 5 for i in range(groups)]
    counts[groups // 3] = 700
    check_experts(counts, 144, 48, torch.bfloat16, period)
