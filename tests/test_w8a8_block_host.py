"""Turning a block's experts into int8 ones, without a GPU."""
import pytest
import torch

from mini_qwen_b200 import Qwen3MoEConfig
from mini_qwen_b200.model.layers import Qwen3MoEBlock


@pytest.mark.parametrize("what", ["bias", "nan"])
def test_a_refused_projection_leaves_the_block_as_it_was(what):
    cfg = Qwen3MoEConfig(hidden_size=32, intermediate_size=16, num_experts=4, num_experts_per_tok=2)
    blk = Qwen3MoEBlock(cfg)
    if what == "bias":
        blk.experts[2].up_proj = torch.nn.Linear(32, 16, bias=True)
    else:
        with torch.no_grad():
            blk.experts[2].up_proj.weight[3, 1] = float("nan")
    before = {k: v.clone() for k, v in blk.state_dict().items()}
    with pytest.raises(ValueError, match="bias" if what == "bias" else "finite"):
        blk.quantize_to_w8a8()
    after = blk.state_dict()
    assert before.keys() == after.keys()
    assert all(torch.equal(before[k].nan_to_num(7.0), after[k].nan_to_num(7.0)) for k in before)
    assert all(isinstance(getattr(ex, p), torch.nn.Linear) for ex in blk.experts for p in ("gate_proj", "up_proj", "down_proj"))
