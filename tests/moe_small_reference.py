"""The whole MoE layer in 64 bits, and how far the two-launch layer may lie from it.

The bound follows the computation.  ``c`` bounds the relative error of a sum by the number of fp32 additions on its longest path
(eight products are added inside an instruction, then a warp's instructions, then 16 warps), each at most one unit in the last
place, 2^-23, of the sum of magnitudes.  From there: errors of g and u move h = silu(g) u (|silu'| < 1.1), h is held to 2^-17
relative (two bf16 numbers; two tf32 numbers are closer), the down sums and the weighted sum add theirs, and the result is
rounded once, half a step of its type."""
import torch

import w8a8_reference as W

UNIT = 2.0 ** -23


def unpack_int4(trio, e, group):
    qw, sc, qz = (t[e] for t in trio)
    q = torch.stack([(qw >> (4 * i)) & 15 for i in range(8)], dim=1).reshape(-1, qw.shape[1]).double()
    z = torch.stack([(qz >> (4 * i)) & 15 for i in range(8)], dim=2).reshape(qz.shape[0], -1).double()
    at = torch.arange(q.shape[0], device=q.device) // group
    return ((q - z[at]) * sc.double()[at]).T


def route(x, router, top_k, bias, renormalize, min_gap=1e-6):
    logits = x.double() @ router.double().T
    if bias is not None:
        logits = logits + bias.double()
    top, ids = torch.sort(logits, dim=1, descending=True, stable=True)
    weights = torch.softmax(top, dim=1)[:, :top_k]
    if renormalize:
        weights = weights / weights.sum(dim=1, keepdim=True)
    return ids[:, :top_k], weights, top


def layer(x, router, experts, top_k, bias=None, renormalize=True, residual=None, int8=False):
    """``experts(e)`` gives (gate [I, H], up [I, H], down [H, I]) in float64.  Returns the output and its bound without the last
    rounding, both float64."""
    ids, weights, _ = route(x, router, top_k, bias, renormalize)
    out = torch.zeros(x.shape, dtype=torch.float64, device=x.device) if residual is None else residual.double()
    bound = out.abs() * UNIT
    rows = x.double()
    if int8:
        q, sx = W.quantize(x)
        rows = q * sx[:, None]
    c = 40 * UNIT
    for e in sorted(set(ids.flatten().tolist())):
        tok, slot = torch.nonzero(ids == e, as_tuple=True)
        gate, up, down = experts(e)
        a = rows[tok]
        g, u = a @ gate.T, a @ up.T
        h = g * torch.sigmoid(g) * u
        dg, du = c * (a.abs() @ gate.abs().T), c * (a.abs() @ up.abs().T)
        if int8:                                   # exact sums, three roundings
            dg, du = 2 * UNIT * g.abs(), 2 * UNIT * u.abs()
        s = (g * torch.sigmoid(g)).abs()
        dh = 1.1 * u.abs() * dg + s * du + 8 * UNIT * h.abs()
        if int8:
            hq, hs = h.abs().amax(1), None
            hs = (hq / 127)[:, None]
            step = torch.where(hs > 0, hs, torch.ones_like(hs))
            v = h / step
            rounded = v.round()
            # an error of h (and of the row's largest) moves v; where that reaches a half, q may be one off
            moved = dh / step + v.abs() * (dh.amax(1, keepdim=True) / (127 * step) + 2 * UNIT)
            near = ((v - rounded).abs() + moved) >= 0.5
            h = rounded * hs
            dh = near.double() * hs + 4 * UNIT * h.abs() + h.abs() * dh.amax(1, keepdim=True) / (127 * step)
        else:
            dh = dh + 2.0 ** -17 * h.abs()
        w = weights[tok, slot][:, None]
        y = h @ down.T
        size = h.abs() @ down.abs().T
        dy = dh @ down.abs().T + c * size
        out = out.index_add(0, tok, w * y)
        # softmax in fp32 of fp32 logits: the logits' error enters the weights as it is
        dw = 2.0 ** -18 * w
        bound = bound.index_add(0, tok, w * dy + dw * y.abs() + (20 * UNIT) * w * size)
    return out, bound


def assert_close(out, ref, bound):
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    fin = torch.isfinite(ref)
    limit = bound + (ref.abs() + bound) * W.half_step(out.dtype) + torch.finfo(out.dtype).smallest_normal
    err = (out.double() - ref).abs()
    assert bool((err <= limit)[fin].all()), (f"off by {float(err[fin].max())}, "
                                             f"{float((err > limit)[fin].double().mean())} of the values")
