"""GPU: h between the two projections of the two-launch layer is an fp32 number.

One expert, a token that picks one column of its weights: g and u are exactly the weights' values, so h = silu(g) u is known to a few
units of fp32.  The down projection takes the difference of two such h, and the residual takes away nearly all of that, so that
the last rounding, to bf16, is a small one.  The two g are chosen such that a sum of two bf16 numbers misses each h by nearly
2^-17, in the direction that adds up."""
import functools

import pytest
import torch

from mini_qwen_b200.kernels import moe_layer_small, w4a16_moe_layer_small

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def as_bf16(v):
    return v.float().to(BF16).double()


@functools.cache
def two_values():
    """(g, u) of two columns, h in 64 bits, and what two bf16 numbers would make of their difference."""
    g = 1.0 + torch.arange(7 * 128).double() / 128
    g = torch.unique(as_bf16(g))
    h = g * torch.sigmoid(g)
    u = 2.0 ** -torch.floor(torch.log2(h))                # a power of two: u changes nothing but the exponent
    h = h * u
    left = h - as_bf16(h)
    left = left - as_bf16(left)
    best = None
    for a in torch.nonzero(left > 0.85 * 2.0 ** -17).flatten().tolist():
        for b in torch.nonzero(left < -0.85 * 2.0 ** -17).flatten().tolist():
            y = h[a] - h[b]
            rounding = (y - as_bf16(y)).abs()             # what the residual leaves
            if best is None or rounding < best[0]:
                best = rounding, a, b
    _, a, b = best
    return g[[a, b]], u[[a, b]], h[[a, b]], float(left[a] - left[b])


def bound(h, out):
    """fp32 all the way.  silu: the exponential is 2 units off (2^-22; it enters with p / (1 + p) < 0.3), the sum half a unit
    (2^-24), the quotient two (2^-22): below 2^-21 of h.  The sums: six products that are not zero, each addition a unit, 2^-23
    of h[0] + h[1] at most; then the residual's, half a unit of the smaller y, and half a step of bf16 of the result."""
    size = float(h.sum())
    return size * (2.0 ** -21 + 6 * 2.0 ** -23) + float((h[0] - h[1]).abs()) * 2.0 ** -24 + float(out.abs()) * 2.0 ** -8


@pytest.mark.parametrize("T", [1, 2, 3, 5, 9, 16])
@pytest.mark.parametrize("kind", ["dense", "w4"])
def test_h_is_held_in_32_bits(kind, T):
    g, u, h, missed = two_values()
    H = I = 128
    at = [5, 90]                                          # columns of h
    x = torch.zeros(T, H, dtype=BF16, device=DEV)
    x[:, 0] = 1
    router = torch.zeros(1, H, dtype=BF16, device=DEV)
    y = h[0] - h[1]
    residual = torch.full((T, H), -float(as_bf16(y)), dtype=BF16, device=DEV)
    if kind == "dense":
        w13, w2 = torch.zeros(1, 2 * I, H, dtype=BF16, device=DEV), torch.zeros(1, H, I, dtype=BF16, device=DEV)
        w13[0, at, 0], w13[0, [I + c for c in at], 0] = g.to(DEV, BF16), u.to(DEV, BF16)
        w2[0, :, at[0]], w2[0, :, at[1]] = 1, -1
        out = moe_layer_small(x, router, w13, w2, 1, residual=residual)
    else:
        def stack(q, scale):                              # zero points 8
            q = q + 8
            words = torch.zeros(q.shape[0] // 8, q.shape[1], dtype=torch.int64)
            for i in range(8):
                words |= q[i::8] << (4 * i)
            words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
            zeros = torch.full((1, q.shape[1] // 8), -0x77777778, dtype=torch.int32)
            return tuple(t.unsqueeze(0).to(DEV) for t in (words, scale.to(BF16).unsqueeze(0), zeros))

        first = torch.zeros(H, I, dtype=torch.int64)
        first[0, at] = 1
        one = torch.ones(I, dtype=torch.float64)
        gate, up = one.clone(), one.clone()
        gate[at], up[at] = g, u
        down = torch.zeros(I, H, dtype=torch.int64)
        down[at[0]], down[at[1]] = 1, -1
        out = w4a16_moe_layer_small(x, router, stack(first, gate), stack(first, up), stack(down, one), 1, residual=residual)
    want = float(y - as_bf16(y))
    limit = bound(h, torch.tensor(want))
    assert missed > 1.5 * limit                           # two bf16 numbers would show
    assert float((out.double() - want).abs().max()) <= limit
