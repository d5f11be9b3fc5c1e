"""The W8A8 operators in 64 bits, from their definition, and how far a result may lie from them."""
import torch


def quantize(x):
    """Rows of x as whole numbers (float64) and their fp32 scales (as float64)."""
    v = x.double()
    scale = (v.abs().amax(-1) / 127).float().double()
    step = torch.where(scale > 0, scale, torch.ones_like(scale))
    q = (v / step[..., None]).round().clamp(-127, 127) * (scale > 0)[..., None]
    bad = ~torch.isfinite(v).all(-1)
    return torch.where(bad[..., None], torch.zeros_like(q), q), torch.where(bad, torch.full_like(scale, float("nan")), scale)


def product(q, sx, w, scales):
    return (q @ w.double().mT) * sx[..., None] * scales.double()


def swiglu(q, sx, w, scales):
    """h in 64 bits and the size of g, which says how much a rounding of g moves silu(g)."""
    g, u = product(q, sx, w, scales).chunk(2, dim=-1)
    return g * torch.sigmoid(g) * u, g.abs()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def assert_close(out, ref, extra=0.0):
    """``out`` against 64 bits: half a step of its type, three fp32 roundings (the sum's conversion and two scales), ``extra``
    relative to the value, and half the smallest number of the type.  NaN in the same places."""
    ref = ref.to(out.device)
    finite = torch.isfinite(ref)
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    rel = half_step(out.dtype) + 3 * 2.0 ** -24 + extra
    bound = ref.abs() * rel + torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps / 2
    err = (out.double() - ref).abs()
    worst = torch.where(finite, err - bound, torch.zeros_like(err))
    assert bool((worst <= 0).all()), f"off by {float(err[finite].max())}, {float((worst > 0).double().mean())} of the values"


def swiglu_extra(g):
    """A relative error d of g moves silu(g) by at most (1 + |g|) d; g and u carry three roundings each (u's are in
    assert_close already): 3 (1 + |g|) 2^-24.  The exponential's argument |g| log2(e) is rounded once and its constant is off by
    half a step, 1.5 * 2^-24 relative, which the exponential turns into 1.5 |g| 2^-24 (together below 5 (1 + |g|) 2^-24).  The
    exponential itself is 2^-22 off, the sum 2^-24, the reciprocal 2^-23 and the three products 2^-24 each: 10 * 2^-24, below
    6 * 2^-23."""
    return (1 + g) * 5 * 2.0 ** -24 + 6 * 2.0 ** -23
