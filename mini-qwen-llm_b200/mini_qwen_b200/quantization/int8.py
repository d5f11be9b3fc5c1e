"""Symmetric int8 quantiser of weights: one scale for each output channel (row of an ``[N, K]`` weight).

A load-time helper like :func:`_per_group_minmax_quantize`; it runs on whatever device the tensor lives on and follows the
arithmetic of the activation kernel (:func:`mini_qwen_b200.kernels.quantize_rows_int8`) bit for bit.
"""
from __future__ import annotations

import torch
from torch import Tensor


def quantize_channels_int8(w: Tensor) -> tuple[Tensor, Tensor]:
    """w [..., N, K] -> (q int8 [..., N, K] in -127..127, scales fp32 [..., N]) with ``w ~ q * scales``.

    scale = max|row| / 127 rounded to fp32, q = round(row / scale) (halves to even); a row of zeros has scale 0.  Weights have
    to be finite."""
    if not torch.is_floating_point(w) or w.dim() < 2:
        raise ValueError("weights to quantise are floating-point [..., N, K]")
    if not bool(torch.isfinite(w).all()):
        raise ValueError("weights to quantise must be finite")
    q = torch.empty(w.shape, dtype=torch.int8, device=w.device)
    scales = torch.empty(w.shape[:-1], dtype=torch.float32, device=w.device)
    if w.numel() == 0:
        return q, scales.zero_()
    # a bounded number of rows at a time: the quotients are taken in 64 bits
    rows, qr, sr = w.reshape(-1, w.shape[-1]), q.view(-1, w.shape[-1]), scales.view(-1)
    step = max(1, (1 << 24) // w.shape[-1])
    for lo in range(0, rows.shape[0], step):
        v = rows[lo:lo + step].double()
        s = (v.abs().amax(dim=-1) / 127.0).float()
        d = s.double().unsqueeze(-1)
        qr[lo:lo + step] = torch.where(d > 0, v / torch.where(d > 0, d, 1.0), 0.0).round().clamp(-127, 127).to(torch.int8)
        sr[lo:lo + step] = s
    return q, scales
