"""The whole MoE layer for a few tokens in two launches: router, top-k, SwiGLU experts, weighted sum, residual.

What :class:`Qwen3MoEBlock` computes (the reference's ``mini_qwen/model/layers/moe.py:49-68``) without the roundings between its
operations: one rounding at the end.  For bf16 and fp16 experts, int4 ones (W4A16) and int8 ones (W8A8); up to 16 tokens."""
from __future__ import annotations

import ctypes

import torch

from .. import _cabi

MAX_TOKENS = 16


def layer_small_supported(layer: _cabi.MoELayer, tokens: int) -> bool:
    """Whether the two-launch call covers ``tokens`` tokens of the layer."""
    return bool(_cabi.load().mq_moe_small_covers(ctypes.addressof(layer), tokens))


def _layer(x, router_weight, inter, top_k, bias, renormalize, group_size=0, int8=False) -> _cabi.MoELayer:
    E, H = router_weight.shape
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (E,) or not bias.is_contiguous()):
        raise ValueError("bias must be contiguous float32 [experts]")
    if not 1 <= top_k <= E:
        raise ValueError(f"top_k must be 1..{E}, got {top_k}")
    return _cabi.MoELayer(hidden=H, inter=inter, experts=E, top_k=top_k, group_size=group_size, dtype=_cabi.dtype_code(x),
                          router_dtype=_cabi.dtype_code(router_weight), renormalize=int(renormalize), int8_experts=int(int8),
                          router=router_weight.data_ptr(), router_bias=None if bias is None else bias.data_ptr())


def _call(layer: _cabi.MoELayer, x, residual, status, index) -> torch.Tensor:
    H = layer.hidden
    if x.shape[-1:] != (H,):
        raise ValueError(f"x must be [..., {H}], got {tuple(x.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("residual must have the shape and dtype of x")
    if status is not None and status.dtype != torch.int32:
        raise ValueError("status is int32 [1]")
    rows = x.contiguous()
    if rows.data_ptr() % 16:                       # a view into a larger buffer: the kernel reads 16 bytes at a time
        rows = rows.clone()
    T = rows.numel() // H
    if residual is not None:
        residual = residual.contiguous()
    out = torch.empty_like(rows)
    if T == 0:
        return out
    lib = _cabi.load()
    address = ctypes.addressof(layer)
    if not lib.mq_moe_small_covers(address, T):
        raise ValueError(f"{T} tokens of this layer (hidden {H}, inter {layer.inter}, {layer.experts} experts, top_k {layer.top_k}) "
                         "are outside what the two-launch layer covers")
    space = lib.mq_moe_small_workspace_bytes(address, T)
    ws = rows.new_empty(space, dtype=torch.uint8)
    rc = _cabi.on_device(index, lib.mq_moe_small, address, rows.data_ptr(), _cabi.ptr(residual), T, ws.data_ptr(), space,
                         out.data_ptr(), _cabi.ptr(status), _cabi.stream_ptr(index))
    if rc:
        _cabi.check(rc, "mq_moe_small")
    _cabi.count_launches(2)
    return out


def _aligned(*tensors):
    for t in tensors:
        if not t.is_contiguous() or t.data_ptr() % 16:
            raise ValueError("expert weights must be contiguous and 16-byte aligned")


def _router(x, router_weight):
    if router_weight.dim() != 2 or 0 in router_weight.shape:
        raise ValueError("router_weight must be [experts, hidden], neither of them 0")
    return router_weight.contiguous()


def moe_layer_small(hidden_states: torch.Tensor, router_weight: torch.Tensor, gate_up_weights: torch.Tensor,
                    down_weights: torch.Tensor, top_k: int = 8, bias: torch.Tensor | None = None, renormalize: bool = True,
                    residual: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """The layer on bf16 or fp16 experts: ``hidden_states`` [..., H] (at most 16 tokens), ``router_weight`` [E, H] (any float
    dtype), ``gate_up_weights`` [E, 2I, H] (gate rows first), ``down_weights`` [E, H, I].

    The ``top_k`` experts with the largest logits (``+ bias``, fp32 [E]; equal ones by ascending id) are weighted by their softmax
    scores, divided by their sum with ``renormalize``.  ``residual`` is added before the one rounding.  ``status`` (int32 [1],
    optional) receives device-side error bits (a bounded wait that ran out)."""
    index = _cabi.one_device(hidden_states, router_weight, gate_up_weights, down_weights, bias, residual, status)
    router_weight = _router(hidden_states, router_weight)
    E, H = router_weight.shape
    if gate_up_weights.dim() != 3 or gate_up_weights.shape[0] != E or gate_up_weights.shape[1] % 2 or gate_up_weights.shape[2] != H:
        raise ValueError(f"gate_up_weights must be [{E}, 2 * inter, {H}], got {tuple(gate_up_weights.shape)}")
    I = gate_up_weights.shape[1] // 2
    if tuple(down_weights.shape) != (E, H, I):
        raise ValueError(f"down_weights must be [{E}, {H}, {I}], got {tuple(down_weights.shape)}")
    if not hidden_states.dtype == gate_up_weights.dtype == down_weights.dtype:
        raise ValueError("activations and weights must share a dtype")
    _aligned(gate_up_weights, down_weights)
    layer = _layer(hidden_states, router_weight, I, top_k, bias, renormalize)
    layer.gate[0], layer.down[0] = gate_up_weights.data_ptr(), down_weights.data_ptr()
    return _call(layer, hidden_states, residual, status, index)


def w4a16_moe_layer_small(hidden_states: torch.Tensor, router_weight: torch.Tensor, gate, up, down, top_k: int = 8,
                          group_size: int = 128, bias: torch.Tensor | None = None, renormalize: bool = True,
                          residual: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`moe_layer_small` on int4 experts: ``gate``, ``up`` and ``down`` are ``(qweight [E, K/8, N], scales [E, K/g, N],
    qzeros [E, K/g, N/8])`` stacks as in :func:`w4a16_grouped_gemm`; bf16, group sizes that are multiples of 128.

    From about six tokens on the block's chain of launches is the faster way for int4 experts (hidden 2048, inter 768, 128
    experts, top-8, in a graph: 23 against 31 us at one token, 51 : 54 at 4, 78 : 70 at 8, 128 : 93 at 16)."""
    index = _cabi.one_device(hidden_states, router_weight, *gate, *up, *down, bias, residual, status)
    router_weight = _router(hidden_states, router_weight)
    E, H = router_weight.shape
    if hidden_states.dtype != torch.bfloat16:
        raise ValueError("activations must be bfloat16")
    if group_size < 128 or group_size % 128:
        raise ValueError(f"group_size must be a multiple of 128, got {group_size}")
    if any(t.dim() != 3 for t in (*gate, *up, *down)):
        raise ValueError("gate, up and down are stacks of experts: (qweight, scales, qzeros), three dimensions each")
    I = gate[0].shape[2]
    for name, trio, kd, n in (("gate", gate, H, I), ("up", up, H, I), ("down", down, I, H)):
        qw, sc, qz = trio
        if (tuple(qw.shape) != (E, kd // 8, n) or tuple(sc.shape) != (E, kd // group_size, n) or kd % group_size or n % 8
                or tuple(qz.shape) != (E, kd // group_size, n // 8) or qw.dtype != torch.int32 or qz.dtype != torch.int32
                or sc.dtype != torch.bfloat16):
            raise ValueError(f"{name} must be int4 stacks of [{E}, {kd}, {n}] with groups of a multiple of 128")
        _aligned(qw)
        if not (sc.is_contiguous() and qz.is_contiguous()) or sc.data_ptr() % 4:
            raise ValueError(f"{name}: scales and zero points must be contiguous, scales 4-byte aligned")
    layer = _layer(hidden_states, router_weight, I, top_k, bias, renormalize, group_size)
    for field, trio in ((layer.gate, gate), (layer.up, up), (layer.down, down)):
        for i, t in enumerate(trio):
            field[i] = t.data_ptr()
    return _call(layer, hidden_states, residual, status, index)


def w8a8_moe_layer_small(hidden_states: torch.Tensor, router_weight: torch.Tensor, gate_up, down, top_k: int = 8,
                         bias: torch.Tensor | None = None, renormalize: bool = True, residual: torch.Tensor | None = None,
                         status: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`moe_layer_small` on int8 experts: ``gate_up`` is (int8 [E, 2I, H], scales fp32 [E, 2I]), ``down`` (int8 [E, H, I],
    scales fp32 [E, H]).  The token rows and the rows of h are quantised to int8 as :func:`quantize_rows_int8` does; bf16, fp16
    or fp32 activations."""
    index = _cabi.one_device(hidden_states, router_weight, *gate_up, *down, bias, residual, status)
    router_weight = _router(hidden_states, router_weight)
    E, H = router_weight.shape
    w13, s13 = gate_up
    w2, s2 = down
    if w13.dim() != 3 or w13.shape[1] % 2:
        raise ValueError("gate and up weights are [E, 2 * I, H]: gate rows, then up rows")
    I = w13.shape[1] // 2
    for name, w, s, shape in (("gate_up", w13, s13, (E, 2 * I, H)), ("down", w2, s2, (E, H, I))):
        if tuple(w.shape) != shape or w.dtype != torch.int8 or tuple(s.shape) != shape[:2] or s.dtype != torch.float32:
            raise ValueError(f"{name} must be int8 {list(shape)} with float32 scales {list(shape[:2])}")
        if not s.is_contiguous():
            raise ValueError(f"{name}: scales must be contiguous")
    _aligned(w13, w2)
    layer = _layer(hidden_states, router_weight, I, top_k, bias, renormalize, int8=True)
    layer.gate[0], layer.gate[1] = w13.data_ptr(), s13.data_ptr()
    layer.down[0], layer.down[1] = w2.data_ptr(), s2.data_ptr()
    return _call(layer, hidden_states, residual, status, index)
