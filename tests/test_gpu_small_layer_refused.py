"""GPU: the block where the two-launch layer's cooperative launch is refused."""
import pytest
import torch

from mini_qwen_b200 import Qwen3MoEConfig, _cabi
from mini_qwen_b200.kernels import w8a8_moe_layer_small
from mini_qwen_b200.model.layers import Qwen3MoEBlock, RMSNorm

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture
def block():
    torch.manual_seed(3)
    cfg = Qwen3MoEConfig(hidden_size=256, intermediate_size=128, num_experts=8, num_experts_per_tok=2)
    blk = Qwen3MoEBlock(cfg).to(DEV).to(torch.bfloat16)
    blk.quantize_to_w8a8()
    return blk


def test_the_chain_computes_what_the_launch_refuses(block, monkeypatch):
    """A process limited to some of the SMs: the call's answer is the library's, given here by a stand-in."""
    x = torch.randn(5, 256, device=DEV).bfloat16()
    norm = RMSNorm(256).to(DEV).to(torch.bfloat16)
    block.small_layer = False
    chain = block(x), block(x, residual=x), block.half_layer(x, norm)
    block.small_layer = None
    few = block(x)
    asked = []
    monkeypatch.setattr(_cabi.load(), "mq_moe_small", lambda *args: asked.append(args) or _cabi.MQ_ERR_NOT_RESIDENT)
    got = block(x), block(x, residual=x), block.half_layer(x, norm)
    assert len(asked) == 1                                # not asked again
    assert all(torch.equal(a, b) for a, b in zip(got, chain)) and not torch.equal(few, chain[0])
    st = block._stacks
    with pytest.raises(RuntimeError, match="share of the GPU"):
        w8a8_moe_layer_small(x, block.gate.weight.data, (st["w13"], st["s13"]), (st["w2"], st["s2"]), 2)


def test_other_failures_are_raised(block, monkeypatch):
    monkeypatch.setattr(_cabi.load(), "mq_moe_small", lambda *args: 4)
    with pytest.raises(RuntimeError, match="launch failed"):
        block(torch.randn(5, 256, device=DEV).bfloat16())
