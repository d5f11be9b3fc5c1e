"""GPU: a few rows times many output channels."""
import pytest
import torch

import w8a8_reference as R
from mini_qwen_b200 import _cabi
from mini_qwen_b200.kernels import w8a8_gemm, w8a8_grouped_swiglu

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("M,K,N,launches", [(1, 2048, 4096, 1), (8, 2048, 4096, 1), (1, 2048, 8192, 1), (4, 2048, 16384, 2),
                                            (8, 1024, 151936, 2), (1, 64, 40000, 2), (16, 16, 16400, 2), (3, 2048, 8195, 1),
                                            (16, 512, 16387, 2), (2, 2064, 33333, 2)])
def test_wide_linears(M, K, N, launches):
    """Every 16 channels quantise the rows again where that is part of the product's launch, so it is not for many channels."""
    g = torch.Generator(device=DEV).manual_seed(N + M)
    x = torch.randn(M, K, generator=g, device=DEV).bfloat16()
    w = torch.randint(-128, 128, (N, K), generator=g, device=DEV, dtype=torch.int8)
    s = torch.rand(N, generator=g, device=DEV) * 0.01 + 1e-4
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    before = _cabi.launch_count
    out = w8a8_gemm(x, w, s, status=status)
    assert _cabi.launch_count - before == launches and status.item() == 0
    q, sx = R.quantize(x)
    R.assert_close(out, R.product(q, sx, w, s))
    assert torch.equal(out, w8a8_gemm(q.to(torch.int8), w, s, x_scale=sx.float()))
    # the library's call without a workspace, or with one that is too small for two launches: the same numbers in one
    lib = _cabi.load()
    for space in (0, 16):
        alone = torch.zeros_like(out)
        ws = torch.empty(max(space, 1), dtype=torch.uint8, device=DEV)
        rc = lib.mq_w8a8_linear_x(x.data_ptr(), 1, K, w.data_ptr(), s.data_ptr(), M, N, K, 1, ws.data_ptr() if space else None, space,
                                  alone.data_ptr(), None, None, _cabi.stream_ptr(0))
        assert rc == 0 and torch.equal(alone, out)


@pytest.mark.parametrize("M,K,N", [(2, 3, 4194240), (2, 3, 4194241), (17, 5, 4200001)])
def test_more_column_tiles_than_a_grid_has_in_one_dimension(M, K, N):
    g = torch.Generator(device=DEV).manual_seed(N + M)
    x = torch.randn(M, K, generator=g, device=DEV).bfloat16()
    w = torch.randint(-128, 128, (N, K), generator=g, device=DEV, dtype=torch.int8)
    s = torch.rand(N, generator=g, device=DEV) * 0.01 + 1e-4
    q, sx = R.quantize(x)
    R.assert_close(w8a8_gemm(x, w, s), R.product(q, sx, w, s))
    h = w8a8_grouped_swiglu(x, w[None, :N // 2 * 2], s[None, :N // 2 * 2] * 0.05, torch.tensor([0, 1, M], dtype=torch.int32, device=DEV))
    ref, size = R.swiglu(q, sx, w[:N // 2 * 2], s[:N // 2 * 2] * 0.05)
    R.assert_close(h, ref, R.swiglu_extra(size))
