"""GPU: arguments that the two-launch layer turns down before it divides by them."""
import pytest
import torch

from mini_qwen_b200.kernels import moe_layer_small, w4a16_moe_layer_small, w8a8_moe_layer_small

pytestmark = pytest.mark.gpu
DEV = "cuda"


def zeros(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype, device=DEV)


def int4(kd, n, group=128):
    return zeros(2, kd // 8, n, dtype=torch.int32), zeros(2, kd // group, n), zeros(2, kd // group, n // 8, dtype=torch.int32)


@pytest.mark.parametrize("group", [0, -128, 1, 64, 129])
def test_group_sizes(group):
    trio = int4(128, 128)
    with pytest.raises(ValueError, match="group_size"):
        w4a16_moe_layer_small(zeros(1, 128), zeros(2, 128), trio, trio, trio, 1, group)


def test_stacks_of_int4_experts_have_three_dimensions():
    trio = int4(128, 128)
    for bad in (tuple(t[0] for t in trio), (trio[0].flatten(), *trio[1:]), (*trio[:2], trio[2][0, 0, 0])):
        for at in range(3):
            with pytest.raises(ValueError, match="dimensions"):
                w4a16_moe_layer_small(zeros(1, 128), zeros(2, 128), *[bad if i == at else trio for i in range(3)], 1)


@pytest.mark.parametrize("experts,hidden", [(2, 0), (0, 16)])
def test_routers_without_experts_or_channels(experts, hidden):
    x, router = zeros(3, hidden), zeros(experts, hidden)
    with pytest.raises(ValueError, match="router_weight"):
        moe_layer_small(x, router, zeros(experts, 32, hidden), zeros(experts, hidden, 16), 1)
    with pytest.raises(ValueError, match="router_weight"):
        w8a8_moe_layer_small(x, router, (zeros(experts, 32, hidden, dtype=torch.int8), zeros(experts, 32, dtype=torch.float32)),
                             (zeros(experts, hidden, 16, dtype=torch.int8), zeros(experts, hidden, dtype=torch.float32)), 1)


def test_experts_without_width():
    with pytest.raises(ValueError):
        moe_layer_small(zeros(1, 16), zeros(2, 16), zeros(2, 0, 16), zeros(2, 16, 0), 1)
