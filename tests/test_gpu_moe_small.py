"""GPU: the whole MoE layer for a few tokens in two launches, against its definition in 64 bits."""
import pytest
import torch

import moe_small_reference as R
from mini_qwen_b200 import _cabi
from mini_qwen_b200.kernels import moe_layer_small, moe_router, w4a16_moe_layer_small, w8a8_moe_layer_small

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class Layer:
    """Experts of one kind, the call on them and its reference."""

    def __init__(self, kind, T, H, I, E, K, dtype=BF16, seed=0, group=128, router_dtype=None):
        g = torch.Generator(device=DEV).manual_seed(1000 * T + H + E + seed)
        self.kind, self.K, self.E, self.I, self.group = kind, K, E, I, group

        def normal(*shape, std=1.0, dt=dtype):
            return (torch.randn(*shape, generator=g, device=DEV) * std).to(dt)

        def bits(*shape):
            return torch.randint(-2 ** 31, 2 ** 31 - 1, shape, generator=g, device=DEV, dtype=torch.int32)

        def int4(kd, n):
            scale = (torch.rand(E, kd // group, n, generator=g, device=DEV) * 0.01 + 0.002).to(BF16)
            return bits(E, kd // 8, n), scale, bits(E, kd // group, n // 8)

        def int8(n, kd):
            return (torch.randint(-128, 128, (E, n, kd), generator=g, device=DEV, dtype=torch.int8),
                    torch.rand(E, n, generator=g, device=DEV) * 4e-4 + 1e-5)

        self.x = normal(T, H)
        self.router = normal(E, H, std=H ** -0.5, dt=router_dtype or dtype)
        if kind == "dense":
            self.w13, self.w2 = normal(E, 2 * I, H, std=H ** -0.5), normal(E, H, I, std=I ** -0.5)
        elif kind == "w4":
            self.trios = int4(H, I), int4(H, I), int4(I, H)
        else:
            self.w13, self.w2 = int8(2 * I, H), int8(H, I)

    def experts(self, e):
        I = self.I
        if self.kind == "dense":
            w = self.w13[e].double()
            return w[:I], w[I:], self.w2[e].double()
        if self.kind == "w4":
            return tuple(R.unpack_int4(t, e, self.group) for t in self.trios)
        w = self.w13[0][e].double() * self.w13[1][e].double()[:, None]
        return w[:I], w[I:], self.w2[0][e].double() * self.w2[1][e].double()[:, None]

    def __call__(self, x=None, **kw):
        x = self.x if x is None else x
        if self.kind == "dense":
            return moe_layer_small(x, self.router, self.w13, self.w2, self.K, **kw)
        if self.kind == "w4":
            return w4a16_moe_layer_small(x, self.router, *self.trios, self.K, self.group, **kw)
        return w8a8_moe_layer_small(x, self.router, self.w13, self.w2, self.K, **kw)

    def check(self, out, x=None, **kw):
        x = self.x if x is None else x
        kw.pop("status", None)
        ref, bound = R.layer(x, self.router, self.experts, self.K, int8=self.kind == "w8", **kw)
        R.assert_close(out, ref, bound)


SHAPES = [(128, 128, 8, 2), (256, 128, 16, 4), (2048, 768, 32, 8), (640, 384, 128, 6), (1024, 256, 5, 5), (256, 256, 300, 3)]
KINDS = [("dense", BF16), ("dense", F16), ("w4", BF16), ("w8", BF16), ("w8", F16), ("w8", F32)]


@pytest.mark.parametrize("T", [1, 2, 7, 8, 9, 16])
@pytest.mark.parametrize("H,I,E,K", SHAPES)
@pytest.mark.parametrize("kind,dtype", KINDS)
def test_layer(kind, dtype, H, I, E, K, T):
    lay = Layer(kind, T, H, I, E, K, dtype)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = lay(status=status)
    assert out.dtype == dtype and out.shape == lay.x.shape and status.item() == 0
    lay.check(out)


@pytest.mark.parametrize("kind,H,I,E,K", [("dense", 8, 8, 1, 1), ("dense", 72, 200, 3, 2), ("dense", 2056, 40, 7, 3),
                                          ("dense", 4096, 1536, 8, 2), ("w8", 16, 16, 2, 2), ("w8", 208, 2000, 3, 1),
                                          ("w8", 4096, 1040, 4, 2), ("w4", 4096, 1280, 4, 2), ("dense", 256, 64, 1024, 32),
                                          ("w8", 256, 64, 1000, 32), ("w4", 128, 128, 1001, 9)])
@pytest.mark.parametrize("T", [1, 5, 16])
def test_odd_layers(kind, H, I, E, K, T):
    lay = Layer(kind, T, H, I, E, K, BF16, seed=1)
    lay.check(lay())


def test_groups_of_256():
    lay = Layer("w4", 6, 512, 256, 8, 2, group=256)
    lay.check(lay())


@pytest.mark.parametrize("group,H,I", [(256, 2048, 768), (384, 1152, 768), (640, 1280, 640)])
def test_larger_groups(group, H, I):
    lay = Layer("w4", 9, H, I, 8, 2, group=group)
    lay.check(lay())


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_options(kind, dtype):
    lay = Layer(kind, 11, 256, 128, 16, 4, dtype, router_dtype=F32 if kind == "w4" else None)
    bias = torch.linspace(-2, 2, 16, device=DEV)
    residual = torch.randn(11, 256, device=DEV, generator=torch.Generator(DEV).manual_seed(2)).to(dtype)
    for kw in ({"bias": bias}, {"renormalize": False}, {"residual": residual},
               {"bias": bias, "renormalize": False, "residual": residual}):
        lay.check(lay(**kw), **kw)
    # shapes with more dimensions, strided rows, rows off the 16-byte grid
    ref = lay()
    assert torch.equal(lay(lay.x.view(1, 11, 256)), ref.view(1, 11, 256))
    wide = torch.zeros(11, 300, dtype=dtype, device=DEV)
    wide[:, 3:259] = lay.x
    assert torch.equal(lay(wide[:, 3:259]), ref)
    flat = torch.zeros(11 * 256 + 1, dtype=dtype, device=DEV)
    flat[1:] = lay.x.flatten()
    assert torch.equal(lay(flat[1:].view(11, 256)), ref)
    assert lay(lay.x[:0]).shape == (0, 256)


@pytest.mark.parametrize("kind", ["dense", "w4", "w8"])
def test_a_token_does_not_depend_on_the_others(kind):
    """Each column of the products is its own, so a batch gives every token what it gets alone, up to the split of the sums."""
    lay = Layer(kind, 16, 512, 256, 8, 3)
    out = lay()
    for t in (0, 7, 8, 15):
        one = lay(lay.x[t:t + 1])
        torch.testing.assert_close(one[0].float(), out[t].float(), rtol=2 ** -7, atol=1e-2)
    assert torch.equal(out, lay())                 # the same bits every time


@pytest.mark.parametrize("kind", ["dense", "w4", "w8"])
def test_all_tokens_on_the_same_experts(kind):
    lay = Layer(kind, 16, 256, 128, 16, 4)
    bias = torch.zeros(16, device=DEV)
    bias[[3, 5, 8, 15]] = 50
    lay.check(lay(bias=bias), bias=bias)


def test_ties_go_to_the_lower_id_and_masked_experts_to_nobody():
    lay = Layer("dense", 9, 256, 128, 16, 3)
    lay.router[9:] = lay.router[2]                 # experts 2, 9, 10, ..., 15 have the same logits
    lay.router[2] *= 1
    bias = torch.zeros(16, device=DEV)
    bias[2] = bias[9:] = 30
    lay.check(lay(bias=bias), bias=bias)           # the reference's stable sort: 2, 9, 10
    lay.router.zero_()                             # all equal: 0, 1, 2
    lay.check(lay())
    bias = torch.full((16,), float("-inf"), device=DEV)
    bias[[4, 11]] = 0
    w = lay.w2.clone()
    lay.w2[[0, 1, 2, 3]] = 1e4                     # what fills up the three places counts for nothing
    out = lay(bias=bias)
    lay.check(out, bias=bias)
    lay.w2 = w


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_infinities_and_nans_stay_where_they_are(kind, dtype):
    lay = Layer(kind, 13, 256, 128, 16, 2, dtype)
    ref = lay()
    x = lay.x.clone()
    x[3, 17] = float("nan")
    x[9, 0] = float("inf")
    x[12] = 0
    out = lay(x)
    rest = [t for t in range(13) if t not in (3, 9, 12)]
    assert torch.equal(out[rest], ref[rest])
    assert torch.isnan(out[3]).all() and not torch.isfinite(out[9]).any() and not out[12].any()
    # weights of experts that a token did not choose do not reach it, whatever they hold
    ids, _ = moe_router(lay.x, lay.router, 2)
    used = torch.bincount(ids.flatten(), minlength=16)
    victim = int(ids[0, 0])
    others = [t for t in range(13) if victim not in ids[t].tolist()]
    assert used[victim] > 0 and others
    if kind == "dense":
        lay.w2[victim] = float("nan")
        lay.w13[victim, 5] = float("inf")
    elif kind == "w4":
        lay.trios[2][1][victim] = float("nan")
    else:
        lay.w2[1][victim] = float("inf")
    out = lay()
    assert torch.equal(out[others], ref[others]) and not torch.isfinite(out[0]).any()


def test_h_beyond_the_range_of_fp16():
    """h is not rounded to the model's type in between: products of 300 x 300 pass fp16's range and come back into it."""
    lay = Layer("dense", 5, 256, 128, 4, 2, F16)
    lay.w13 *= 300
    lay.w2 *= 1e-3
    out = lay()
    assert torch.isfinite(out).all()
    lay.check(out)


def test_overlapping_calls_and_graphs():
    """Every call has a workspace of its own: calls on several streams and graphs replayed at the same time do not meet."""
    lays = [Layer("dense", 8, 2048, 768, 16, 4, seed=s) for s in range(2)] + [Layer("w8", 16, 1024, 512, 16, 4, seed=3)]
    refs = [lay() for lay in lays]
    streams = [torch.cuda.Stream() for _ in lays]
    torch.cuda.synchronize()
    outs = [[] for _ in lays]
    for _ in range(10):
        for i, (lay, st) in enumerate(zip(lays, streams)):
            with torch.cuda.stream(st):
                outs[i].append(lay())
    torch.cuda.synchronize()
    for got, ref in zip(outs, refs):
        assert all(torch.equal(o, ref) for o in got)
    graphs, held = [], []
    for lay in lays:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(lay())
        graphs.append(graph)
    for _ in range(10):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for out, ref in zip(held, refs):
        assert torch.equal(out, ref)


def test_refusals():
    lay = Layer("dense", 4, 128, 128, 8, 2)
    w4, w8 = Layer("w4", 4, 128, 128, 8, 2), Layer("w8", 4, 128, 128, 8, 2)
    x = lay.x
    bad = [lambda: lay(torch.zeros(17, 128, dtype=BF16, device=DEV)), lambda: lay(x.half()), lambda: lay(x[:, :64]),
           lambda: lay(x.cpu()), lambda: lay(bias=torch.zeros(7, device=DEV)), lambda: lay(bias=torch.zeros(8, dtype=BF16, device=DEV)),
           lambda: lay(residual=x[:2]), lambda: lay(residual=x.float()),
           lambda: moe_layer_small(x, lay.router, lay.w13[:, :-1], lay.w2, 2),
           lambda: moe_layer_small(x, lay.router, lay.w13, lay.w2[:, :, :64], 2),
           lambda: moe_layer_small(x, lay.router, lay.w13, lay.w2, 9), lambda: moe_layer_small(x, lay.router, lay.w13, lay.w2, 0),
           lambda: moe_layer_small(x, lay.router, lay.w13.transpose(1, 2).contiguous().transpose(1, 2), lay.w2, 2),
           lambda: moe_layer_small(x.float(), lay.router.float(), lay.w13.float(), lay.w2.float(), 2),
           lambda: w4(w4.x.half()), lambda: w4a16_moe_layer_small(w4.x, w4.router, *w4.trios, 2, 64),
           lambda: w8a8_moe_layer_small(w8.x, w8.router, (w8.w13[0], w8.w13[1].half()), w8.w2, 2),
           lambda: w8a8_moe_layer_small(w8.x, w8.router, w8.w13, (w8.w2[0].transpose(1, 2), w8.w2[1]), 2)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    big = _cabi.MoELayer(hidden=128, inter=16384, experts=8, top_k=8, dtype=1, router_dtype=1, int8_experts=1)
    import ctypes
    lib = _cabi.load()
    assert lib.mq_moe_small_covers(ctypes.addressof(big), 16) == 1 and lib.mq_moe_small_covers(ctypes.addressof(big), 17) == 0
    # a workspace that is too small, or not there, is refused before any launch
    big.inter, big.int8_experts = 128, 0
    big.router, big.gate[0], big.down[0] = lay.router.data_ptr(), lay.w13.data_ptr(), lay.w2.data_ptr()
    big.top_k = 2
    out = torch.empty_like(x)
    args = (x.data_ptr(), None, 4)
    assert lib.mq_moe_small(ctypes.addressof(big), *args, out.data_ptr(), 100, out.data_ptr(), None, None) == 3
    assert lib.mq_moe_small(ctypes.addressof(big), *args, None, 1 << 20, out.data_ptr(), None, None) == 1
