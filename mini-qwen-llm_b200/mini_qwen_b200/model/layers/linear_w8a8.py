"""W8A8 linear layer, beside :class:`LinearW4A16`: int8 weights with a scale for each output channel, activations quantised to
int8 with a scale for each token as they come."""
from __future__ import annotations

import torch
import torch.nn as nn

from ...kernels.w8a8_gemm import w8a8_gemm
from ...quantization.int8 import quantize_channels_int8


class LinearW8A8(nn.Module):
    """``y = q(x) @ qweight.T * scales`` in the type of x (bf16, fp16 or fp32).

    Buffers: ``qweight`` int8 [N, K] (the layout of ``nn.Linear.weight``), ``scales`` fp32 [N].  ``module.to(dtype)`` must not
    touch the scales, so they stay fp32 (see ``_apply``)."""

    _status = None     # device status word, allocated by the first call

    def __init__(self, in_features: int, out_features: int):
        super().__init__()
        self.in_features = in_features
        self.out_features = out_features
        self.register_buffer("qweight", torch.zeros(out_features, in_features, dtype=torch.int8))
        self.register_buffer("scales", torch.zeros(out_features, dtype=torch.float32))

    def _apply(self, fn, *args, **kwargs):
        scales = self.scales
        super()._apply(fn, *args, **kwargs)
        if self.scales.dtype != torch.float32:      # .half(), .to(torch.bfloat16): the scales only change their device
            self.scales = scales.to(self.scales.device)
        return self

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        rows = x if x.dim() == 2 and x.shape[1] == self.in_features else x.reshape(-1, self.in_features)
        status = None
        if rows.is_cuda:       # which calls take a kernel with bounded waits goes by rows, sizes and alignment
            status = self._status
            if status is None or status.device != rows.device:
                status = self._status = torch.zeros(1, dtype=torch.int32, device=rows.device)
        y = w8a8_gemm(rows, self.qweight, self.scales, status=status)
        return y if rows is x else y.reshape(*x.shape[:-1], self.out_features)

    def check_status(self) -> None:
        """Raises if a kernel of this layer reported a device-side error (synchronises)."""
        if self._status is not None and int(self._status.item()) & 1:
            raise RuntimeError("a bounded wait expired inside a W8A8 kernel; the last output is invalid")

    @classmethod
    def from_float(cls, linear: nn.Linear) -> "LinearW8A8":
        """Quantise an ``nn.Linear`` (weight [N, K], no bias) channel by channel, on the weight's device."""
        if linear.bias is not None:
            raise ValueError("LinearW8A8 has no bias; add it to the result")
        with torch.no_grad():
            qweight, scales = quantize_channels_int8(linear.weight.data)
        with torch.device("meta"):
            layer = cls(qweight.shape[1], qweight.shape[0])
        layer.qweight, layer.scales = qweight, scales
        return layer

    def extra_repr(self) -> str:
        return f"in={self.in_features}, out={self.out_features}"
