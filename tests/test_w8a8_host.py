"""W8A8 without a GPU: the weight quantiser, the layer's buffers, refusals."""
import pytest
import torch

from mini_qwen_b200 import _cabi
from mini_qwen_b200.kernels import quantize_rows_int8, w8a8_gemm, w8a8_grouped_gemm, w8a8_grouped_swiglu
from mini_qwen_b200 import Qwen3MoEConfig
from mini_qwen_b200.model.layers import LinearW8A8, Qwen3MoEBlock
from mini_qwen_b200.quantization import quantize_channels_int8
import w8a8_reference as R


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_channel_quantiser_follows_the_definition(dtype):
    w = torch.randn(3, 7, 65, generator=torch.Generator().manual_seed(1)).to(dtype)
    w[1, 2] = 0
    w[0, 0] = torch.linspace(-127, 127, 65)          # scale 1: quotients that are halves exactly, to even
    q, s = quantize_channels_int8(w)
    rq, rs = R.quantize(w)
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and q.shape == w.shape and s.shape == (3, 7)
    assert torch.equal(q.double(), rq) and torch.equal(s.double(), rs)
    assert s[1, 2] == 0 and not q[1, 2].any()


def test_channel_quantiser_refuses_what_has_no_scale():
    for bad in (float("inf"), float("nan")):
        with pytest.raises(ValueError, match="finite"):
            quantize_channels_int8(torch.tensor([[1.0, bad]]))
    with pytest.raises(ValueError):
        quantize_channels_int8(torch.zeros(2, 2, dtype=torch.int8))


def test_linear_w8a8_keeps_its_scales_in_fp32():
    lin = torch.nn.Linear(48, 40, bias=False)
    layer = LinearW8A8.from_float(lin)
    assert sorted(layer.state_dict()) == ["qweight", "scales"]
    before = layer.scales.clone()
    layer = layer.to(torch.bfloat16)
    assert layer.scales.dtype == torch.float32 and torch.equal(layer.scales, before)
    assert layer.qweight.dtype == torch.int8
    back = layer.qweight.double() * layer.scales.double()[:, None]
    assert ((back - lin.weight.double()).abs() <= layer.scales.double()[:, None] * 0.5000001).all()
    fresh = LinearW8A8(48, 40)
    fresh.load_state_dict(layer.state_dict())
    assert torch.equal(fresh.qweight, layer.qweight)
    with pytest.raises(ValueError, match="bias"):
        LinearW8A8.from_float(torch.nn.Linear(8, 8))


def test_cpu_tensors_are_refused():
    x, w, s = torch.zeros(2, 16), torch.zeros(8, 16, dtype=torch.int8), torch.zeros(8)
    off = torch.tensor([0, 2], dtype=torch.int32)
    for call in (lambda: quantize_rows_int8(x), lambda: w8a8_gemm(x, w, s), lambda: w8a8_grouped_gemm(x, w[None], s[None], off),
                 lambda: w8a8_grouped_swiglu(x, w[None], s[None], off), lambda: LinearW8A8(16, 8)(x)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_c_calls_check_their_arguments():
    lib = _cabi.load()
    one = 4096                                        # never dereferenced: every call below returns before a launch
    assert lib.mq_quantize_rows_int8(one, 1, -1, 8, 8, one, one, None) == 1
    assert lib.mq_quantize_rows_int8(one, 7, 1, 8, 8, one, one, None) == 1
    assert lib.mq_quantize_rows_int8(None, 1, 1, 8, 8, one, one, None) == 1
    assert lib.mq_quantize_rows_int8(one, 1, 1 << 31, 8, 8, one, one, None) == 2
    assert lib.mq_quantize_rows_int8(None, 1, 0, 8, 8, None, None, None) == 0
    assert lib.mq_w8a8_linear(one, one, one, one, 1, 8, 131072, 1, one, None, None) == 2
    assert lib.mq_w8a8_linear(one, one, one, one, 1, 8, 16, 9, one, None, None) == 1
    assert lib.mq_w8a8_linear(one, None, one, one, 1, 8, 16, 1, one, None, None) == 1
    assert lib.mq_w8a8_linear(None, None, None, None, 0, 8, 16, 1, None, None, None) == 0
    assert lib.mq_w8a8_grouped_gemm(one, one, one, one, None, 4, 2, 2, 8, 16, 1, one, None, None) == 1
    assert lib.mq_w8a8_grouped_gemm(one, one, one, one, one, 4, 2, 3, 8, 16, 1, one, None, None) == 1
    assert lib.mq_w8a8_grouped_swiglu(one, one, None, 3, 1, one, one, one, 4, 2, 2, 8, 16, 1, one, None, None) == 1
    assert lib.mq_w8a8_grouped_swiglu(one, one, one, 0, 1, one, one, one, 4, 2, 2, 8, 16, 1, one, None, None) == 1
    assert lib.mq_w8a8_grouped_swiglu(one, one, one, 3, 0, one, one, one, 4, 2, 2, 8, 16, 1, one, None, None) == 1


def _block(**kw):
    cfg = Qwen3MoEConfig(hidden_size=64, intermediate_size=32, num_experts=4, num_experts_per_tok=2)
    return cfg, Qwen3MoEBlock(cfg, **kw)


def test_block_swaps_its_projections_for_int8_ones():
    cfg, blk = _block()
    want = quantize_channels_int8(blk.experts[2].up_proj.weight.data)
    blk.quantize_to_w8a8()
    lin = blk.experts[2].up_proj
    assert isinstance(lin, LinearW8A8) and torch.equal(lin.qweight, want[0]) and torch.equal(lin.scales, want[1])
    blk.finalize()
    assert blk._stacks["w13"].shape == (4, 64, 64) and blk._stacks["s13"].shape == (4, 64)
    assert torch.equal(blk._stacks["w13"][2, 32:], want[0]) and torch.equal(blk._stacks["s13"][2, 32:], want[1])
    other = Qwen3MoEBlock.from_stacked_w8(cfg, blk.gate.weight.data, (blk._stacks["w13"], blk._stacks["s13"]),
                                          (blk._stacks["w2"], blk._stacks["s2"]))
    a, b = blk.state_dict(), other.state_dict()
    assert a.keys() == b.keys() and all(torch.equal(a[k], b[k]) for k in a)
    with pytest.raises(ValueError):
        blk.quantize_to_w8a8()                      # quantised already


def test_block_refuses_mixed_experts_and_wrong_stacks():
    cfg, blk = _block()
    blk.experts[1].down_proj = LinearW8A8.from_float(blk.experts[1].down_proj)
    with pytest.raises(ValueError):
        blk.finalize()
    q = torch.zeros(4, 64, 64, dtype=torch.int8), torch.zeros(4, 64)
    d = torch.zeros(4, 64, 32, dtype=torch.int8), torch.zeros(4, 64)
    for bad in ((q, (d[0], d[1][:, :32])), ((q[0][:3], q[1]), d), ((q[0].float(), q[1]), d)):
        with pytest.raises(ValueError):
            Qwen3MoEBlock.from_stacked_w8(cfg, blk.gate.weight.data, *bad)
