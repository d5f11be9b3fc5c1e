"""GPU: the block on int8 experts, and the two-launch layer as the block calls it."""
import pytest
import torch

import moe_small_reference as R
import w8a8_reference as W
from mini_qwen_b200 import Qwen3MoEConfig
from mini_qwen_b200.graph import CapturedForward
from mini_qwen_b200.kernels import (moe_permute_plan, moe_router, moe_unpermute, w8a8_grouped_gemm, w8a8_grouped_swiglu_gather)
from mini_qwen_b200.model.layers import LinearW8A8, Qwen3MoEBlock, RMSNorm
from mini_qwen_b200.quantization import quantize_channels_int8

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def make(dtype=BF16, H=256, I=128, E=16, K=4, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    cfg = Qwen3MoEConfig(hidden_size=H, intermediate_size=I, num_experts=E, num_experts_per_tok=K)
    router = (torch.randn(E, H, generator=g, device=DEV) * H ** -0.5).to(dtype)
    w13 = torch.randn(E, 2 * I, H, generator=g, device=DEV) * H ** -0.5
    w2 = torch.randn(E, H, I, generator=g, device=DEV) * I ** -0.5
    dense = Qwen3MoEBlock.from_stacked(cfg, router, w13.to(dtype), w2.to(dtype))
    q13, q2 = quantize_channels_int8(w13.to(dtype)), quantize_channels_int8(w2.to(dtype))
    return cfg, router, dense, q13, q2, g


def rows(g, T, H, dtype):
    return torch.randn(T, H, generator=g, device=DEV).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T", [1, 16, 17, 64, 65, 300])
def test_block_is_the_chain_of_its_functions(dtype, T):
    """Over 16 tokens the block's call is, bit for bit, the functions one after the other."""
    cfg, router, _, q13, q2, g = make(dtype)
    blk = Qwen3MoEBlock.from_stacked_w8(cfg, router, q13, q2)
    x = rows(g, T, 256, dtype)
    ids, w = moe_router(x, router, 4, renormalize=True)
    perm, inv, off, _ = moe_permute_plan(ids.to(torch.int32), 16, want_int64_offsets=False)
    h = w8a8_grouped_swiglu_gather(x, perm, 4, *q13, off)
    ref = moe_unpermute(w8a8_grouped_gemm(h, *q2, off), w, ids, T)
    if T <= 16:
        small = blk(x)
        layer = lambda e: (q13[0][e, :128].double() * q13[1][e, :128].double()[:, None],      # noqa: E731
                           q13[0][e, 128:].double() * q13[1][e, 128:].double()[:, None],
                           q2[0][e].double() * q2[1][e].double()[:, None])
        R.assert_close(small, *R.layer(x, router, layer, 4, int8=True))
        blk.small_layer = False
    out = blk(x)
    blk.check_status()
    # the routing of a small batch sums the logits in another order: weights may differ in the last place
    if T > 64:
        assert torch.equal(out, ref)
    tol = {BF16: 2.0 ** -7, F16: 2.0 ** -10, F32: 2.0 ** -18}[dtype]
    torch.testing.assert_close(out.float(), ref.float(), rtol=tol, atol=tol)
    blk.kernel_events = []                           # stage by stage
    torch.testing.assert_close(blk(x).float(), ref.float(), rtol=tol, atol=tol)
    assert "grouped_swiglu" in [name for name, *_ in blk.kernel_events]


def test_quantised_block_stays_close_to_the_dense_one():
    """Each quantisation is off by half a step: with 256 and 128 products of random sign the output's error stays within a few
    percent of its size (half a step of a row of 256 normal numbers is 3 / 254 of their deviation, two rows and two products
    make about 2 %)."""
    cfg, router, dense, *_, g = make(BF16)
    x = rows(g, 40, 256, BF16)
    ref = dense(x).float()
    dense.quantize_to_w8a8()
    assert all(isinstance(getattr(ex, p), LinearW8A8) for ex in dense.experts for p in ("gate_proj", "up_proj", "down_proj"))
    out = dense(x).float()
    assert float((out - ref).norm() / ref.norm()) < 0.05
    few = dense(x[:8]).float()                       # in two launches
    assert float((few - out[:8]).norm() / out[:8].norm()) < 0.01


def test_stacks_are_views_and_follow_a_swapped_projection():
    cfg, router, dense, q13, q2, g = make(BF16)
    dense.quantize_to_w8a8()
    x = rows(g, 30, 256, BF16)
    first = dense(x)
    st = dense._stacks
    assert dense.experts[3].up_proj.qweight.data_ptr() == st["w13"][3, 128:].data_ptr()
    assert dense.experts[3].down_proj.scales.data_ptr() == st["s2"][3].data_ptr()
    built = Qwen3MoEBlock.from_stacked_w8(cfg, router, q13, q2)
    assert torch.equal(built(x), first)
    state = {k: v.clone() for k, v in dense.state_dict().items()}
    assert state["experts.0.gate_proj.qweight"].dtype == torch.int8 and state["experts.0.gate_proj.scales"].dtype == F32
    dense.experts[5].down_proj = LinearW8A8.from_float(torch.nn.Linear(128, 256, bias=False).to(DEV))
    assert not torch.equal(dense(x), first)
    dense.load_state_dict(state)
    assert torch.equal(dense(x), first)
    dense = dense.to(torch.float16)                  # activations of another type; scales stay fp32
    assert dense.experts[0].gate_proj.scales.dtype == F32
    assert dense(x.half()).dtype == F16
    dense.experts[1].up_proj = torch.nn.Linear(256, 128, bias=False).to(DEV)
    with pytest.raises(ValueError, match="mix"):
        dense(x.half())


@pytest.mark.parametrize("T", [1, 7, 50])
def test_half_layer_and_graph(T):
    cfg, router, _, q13, q2, g = make(BF16)
    blk = Qwen3MoEBlock.from_stacked_w8(cfg, router, q13, q2)
    norm = RMSNorm(256).to(DEV).to(BF16)
    norm.weight.data.uniform_(0.5, 1.5)
    h = rows(g, T, 256, BF16)
    out = blk.half_layer(h, norm)
    ref = blk(norm(h), residual=h)
    assert torch.equal(out, ref)
    torch.testing.assert_close(out.float(), h.float() + blk(norm(h)).float(), rtol=2 ** -6, atol=2 ** -6)
    cap = CapturedForward(lambda x: blk.half_layer(x, norm), h)
    for seed in range(3):
        h2 = rows(g, T, 256, BF16)
        cap.x.copy_(h2)
        assert torch.equal(cap.replay(), blk.half_layer(h2, norm))
    blk.check_status()


@pytest.mark.parametrize("kind", ["dense", "w4"])
def test_the_two_launch_layer_is_the_blocks_choice_to_make(kind):
    """Off by default for dense and int4 experts, whose call keeps its results; on by a flag, and close to the chain: the
    chain rounds g, silu(g), u, their product and the expert's output to bf16, half a step (2^-9) each, and the weights' sum
    once more."""
    cfg, router, blk, *_, g = make(BF16, H=256, I=256)
    if kind == "w4":
        blk.quantize_to_w4a16(128)
    x = rows(g, 11, 256, BF16)
    chain = blk(x)
    assert blk.small_layer is None
    blk.small_layer = True
    small = blk(x)
    err = (small.double() - chain.double()).abs()
    assert float(err.max()) <= 8 * 2.0 ** -9 * float(chain.abs().max()) and not torch.equal(small, chain)
    many = rows(g, 17, 256, BF16)
    blk.small_layer = False
    ref = blk(many), blk(x)
    assert torch.equal(ref[1], chain)
    blk.small_layer = True
    assert torch.equal(blk(many), ref[0])            # more than 16 tokens: the chain
    # a view off the 16-byte grid is copied first, on either path
    flat = torch.zeros(11 * 256 + 1, dtype=BF16, device=DEV)
    flat[1:] = x.flatten()
    assert torch.equal(blk(flat[1:].view(11, 256)), small)
    blk.small_layer = False
    assert torch.equal(blk(flat[1:].view(11, 256)), chain)
    blk.check_status()


def test_layers_in_a_row():
    """Prefill and decode steps through three W8A8 layers, eager and as one graph: a row's result does not depend on how it is
    replayed, and follows the dense layers as closely as three quantised layers can."""
    layers = []
    for seed in range(3):
        _, _, dense, q13, q2, g = make(BF16, seed=seed)
        cfg, router = dense.config if hasattr(dense, "config") else make(BF16, seed=seed)[0], dense.gate.weight.data
        norm = RMSNorm(256).to(DEV).to(BF16)
        norm.weight.data.uniform_(0.8, 1.2)
        layers.append((Qwen3MoEBlock.from_stacked_w8(cfg, router, q13, q2), dense, norm))

    def run(h, which):
        for layer in layers:
            h = layer[which].half_layer(h, layer[2])
        return h

    for T in (33, 2, 1, 16, 17):
        h = rows(g, T, 256, BF16)
        out, ref = run(h, 0), run(h, 1)
        # 2 % of a layer's addition to the residual, three times (see test_quantised_block_stays_close_to_the_dense_one)
        assert float((out - ref).float().norm() / (ref - h).float().norm()) < 0.1
        cap = CapturedForward(lambda x: run(x, 0), h)
        for _ in range(2):
            h2 = rows(g, T, 256, BF16)
            cap.x.copy_(h2)
            assert torch.equal(cap.replay(), run(h2, 0))
    for layer in layers:
        layer[0].check_status()
