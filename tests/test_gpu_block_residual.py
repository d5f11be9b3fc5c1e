"""GPU: the block's residual as a view into a larger buffer."""
import pytest
import torch

from mini_qwen_b200 import Qwen3MoEConfig
from mini_qwen_b200.model.layers import Qwen3MoEBlock, RMSNorm

pytestmark = pytest.mark.gpu
DEV = "cuda"


def off_the_grid(t):
    flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device=DEV)
    flat[1:] = t.flatten()
    return flat[1:].view(t.shape)


@pytest.mark.parametrize("kind", ["dense", "w4", "w8"])
@pytest.mark.parametrize("T", [3, 40])
def test_a_residual_off_the_16_byte_grid(kind, T):
    torch.manual_seed(T)
    cfg = Qwen3MoEConfig(hidden_size=256, intermediate_size=128, num_experts=8, num_experts_per_tok=2)
    blk = Qwen3MoEBlock(cfg).to(DEV).to(torch.bfloat16)
    norm = RMSNorm(256).to(DEV).to(torch.bfloat16)
    if kind != "dense":
        blk.quantize_to_w4a16(128) if kind == "w4" else blk.quantize_to_w8a8()
    x, res = (torch.randn(T, 256, device=DEV).bfloat16() for _ in range(2))
    for small in (None, False):
        blk.small_layer = small
        assert torch.equal(blk(x, residual=off_the_grid(res)), blk(x, residual=res))
        assert torch.equal(blk(off_the_grid(x), residual=off_the_grid(res)), blk(x, residual=res))
        wide = torch.zeros(T, 300, dtype=torch.bfloat16, device=DEV)
        wide[:, 5:261] = res
        assert torch.equal(blk(x, residual=wide[:, 5:261]), blk(x, residual=res))
        assert torch.equal(blk.half_layer(off_the_grid(x), norm), blk.half_layer(x, norm))
    blk.kernel_events = []                                # stage by stage
    assert torch.equal(blk(x, residual=off_the_grid(res)), blk(x, residual=res))
