"""W8A8 products: int8 weights with a scale for each output channel, int8 activations with a scale for each token.

The reference has no 8-bit path; the calls stand beside :mod:`.w4a16_gemm` and :mod:`.moe_grouped_gemm` and follow their shapes.
Activations are given as bf16, fp16 or fp32 rows, which the call quantises itself, or as int8 rows together with their scales
(``x_scale``, from :func:`quantize_rows_int8`) where several products read the same rows."""
from __future__ import annotations

import torch

from .. import _cabi
from .w4a16_gemm import _offsets32

MAX_K = 131071      # 128 * 128 * K < 2^31: the int32 sums are exact


def quantize_rows_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., K] -> (q int8 [..., K] in -127..127, scale fp32 [...]): ``scale = max|row| / 127`` rounded to fp32 and
    ``q = round(row / scale)``, halves to even.  A row of zeros has scale 0; a row that holds an infinity or a NaN has scale NaN
    and q 0, so that what is computed from it is NaN.  Rows may lie apart (a slice of wider rows is read in place)."""
    device = _cabi.one_device(x)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError("rows to quantise are [..., K] with K >= 1")
    code = _cabi.dtype_code(x)
    K = x.shape[-1]
    rows = x if x.dim() == 2 else x.reshape(-1, K)
    if rows.stride(1) != 1 and K > 1 or rows.stride(0) < 0:
        rows = rows.contiguous()
    q = torch.empty(x.shape, dtype=torch.int8, device=device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=device)
    T = rows.shape[0]
    with _cabi.current_device(device):
        rc = _cabi.load().mq_quantize_rows_int8(rows.data_ptr(), code, T, K, rows.stride(0), q.data_ptr(), scale.data_ptr(),
                                                _cabi.stream_ptr(device))
    _cabi.check(rc, "mq_quantize_rows_int8")
    _cabi.count_launches(1 if T else 0)
    return q, scale


def _check_weight(qweight, scales, lead: int):
    if qweight.dtype != torch.int8 or scales.dtype != torch.float32:
        raise ValueError("weights are int8 with float32 scales")
    if qweight.dim() != lead + 2 or scales.shape != qweight.shape[:-1]:
        raise ValueError(f"weights are {'[E, N, K]' if lead else '[N, K]'} with a scale for each output channel; got "
                         f"{tuple(qweight.shape)} and {tuple(scales.shape)}")
    if not 1 <= qweight.shape[-1] <= MAX_K:
        raise ValueError(f"K must be 1..{MAX_K}, got {qweight.shape[-1]}")
    if qweight.shape[-2] == 0 or lead and qweight.shape[0] == 0:
        raise ValueError("the weights have no output channels")


def _rows(x, x_scale, K, out_dtype):
    """The int8 rows, their scales and the type of the result."""
    if x.dim() != 2 or x.shape[1] != K:
        raise ValueError(f"activations are [rows, {K}], got {tuple(x.shape)}")
    if x.dtype == torch.int8:
        if x_scale is None or x_scale.dtype != torch.float32 or x_scale.shape != x.shape[:1]:
            raise ValueError("int8 activations come with x_scale, float32 [rows]")
        return x.contiguous(), x_scale.contiguous(), torch.bfloat16 if out_dtype is None else out_dtype
    if x_scale is not None:
        raise ValueError("x_scale belongs to int8 activations")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    q, scale = quantize_rows_int8(x)
    return q, scale, out_dtype


def _out_code(out_dtype) -> int:
    if out_dtype not in _cabi._DTYPES:
        raise ValueError(f"unsupported result dtype {out_dtype}; expected float32, bfloat16 or float16")
    return _cabi._DTYPES[out_dtype]


def w8a8_gemm(x: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor, x_scale: torch.Tensor | None = None,
              out_dtype: torch.dtype | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """``(q @ qweight.T) * x_scale[:, None] * scales`` with q and x_scale the int8 rows of x; [M, N].

    x [M, K] bf16, fp16 or fp32, or int8 with ``x_scale`` [M]; qweight int8 [N, K]; scales fp32 [N].  The result has x's type
    (bf16 for int8 rows) unless ``out_dtype`` says otherwise.  ``status`` (int32 [1], optional) receives device-side error bits
    (a bounded wait that ran out)."""
    device = _cabi.one_device(x, qweight, scales, x_scale, status)
    _check_weight(qweight, scales, 0)
    N, K = qweight.shape
    q, sx, out_dtype = _rows(x, x_scale, K, out_dtype)
    code = _out_code(out_dtype)
    qweight, scales = qweight.contiguous(), scales.contiguous()
    M = q.shape[0]
    out = torch.empty(M, N, dtype=out_dtype, device=device)
    with _cabi.current_device(device):
        rc = _cabi.load().mq_w8a8_linear(q.data_ptr(), sx.data_ptr(), qweight.data_ptr(), scales.data_ptr(), M, N, K, code,
                                         out.data_ptr(), _cabi.ptr(status), _cabi.stream_ptr(device))
    _cabi.check(rc, "mq_w8a8_linear")
    _cabi.count_launches(1 if M else 0)
    return out


def _groups(expert_offsets, E: int) -> int:
    if expert_offsets.dim() != 1 or expert_offsets.dtype not in (torch.int32, torch.int64):
        raise ValueError("expert_offsets are one-dimensional int32 or int64")
    groups = expert_offsets.numel() - 1
    if groups < E or groups % E:
        raise ValueError(f"expert_offsets hold {groups} groups; the weights hold {E} experts")
    return groups


def _prepare(offsets, S: int, groups: int, N: int, out, code: int):
    """Zeros in the rows of ``out`` (if given) that no group covers, and int32 offsets: one launch where either is due."""
    wide = offsets.dtype == torch.int64
    offsets = offsets.contiguous()
    if out is None and not wide or S == 0:
        return _offsets32(offsets)
    narrow = torch.empty(groups + 1, dtype=torch.int32, device=offsets.device) if wide else offsets
    rc = _cabi.load().mq_grouped_prepare(offsets.data_ptr(), int(wide), S, groups, N, code, _cabi.ptr(out),
                                         narrow.data_ptr() if wide else None, None, _cabi.stream_ptr(offsets.device))
    _cabi.check(rc, "mq_grouped_prepare")
    _cabi.count_launches(1)
    return narrow


def w8a8_grouped_gemm(x: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor, expert_offsets: torch.Tensor,
                      x_scale: torch.Tensor | None = None, zero_init: bool = True, out: torch.Tensor | None = None,
                      out_dtype: torch.dtype | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`w8a8_gemm` of rows ``offsets[e]:offsets[e+1]`` with the weight of expert e.

    qweight int8 [E, N, K], scales fp32 [E, N], offsets [E+1] ascending (or G * E groups, group g on expert g % E).  Rows that no
    group covers are zero (``zero_init=False``: unwritten); with ``out`` given they keep what they hold."""
    device = _cabi.one_device(x, qweight, scales, expert_offsets, x_scale, out, status)
    _check_weight(qweight, scales, 1)
    E, N, K = qweight.shape
    groups = _groups(expert_offsets, E)
    if out is not None:
        if out_dtype is not None and out.dtype != out_dtype:
            raise ValueError("out and out_dtype differ")
        out_dtype = out.dtype
        if tuple(out.shape) != (x.shape[0], N) or not out.is_contiguous():
            raise ValueError(f"out must be contiguous [{x.shape[0]}, {N}]")
    with _cabi.current_device(device):
        q, sx, out_dtype = _rows(x, x_scale, K, out_dtype)
        code = _out_code(out_dtype)
        S = q.shape[0]
        zero = out is None and zero_init
        if out is None:
            out = torch.empty(S, N, dtype=out_dtype, device=device)
        qweight, scales = qweight.contiguous(), scales.contiguous()
        offsets = _prepare(expert_offsets, S, groups, N, out if zero else None, code)
        rc = _cabi.load().mq_w8a8_grouped_gemm(q.data_ptr(), sx.data_ptr(), qweight.data_ptr(), scales.data_ptr(),
                                               offsets.data_ptr(), S, groups, E, N, K, code, out.data_ptr(),
                                               _cabi.ptr(status), _cabi.stream_ptr(device))
    _cabi.check(rc, "mq_w8a8_grouped_gemm")
    _cabi.count_launches(1 if S else 0)
    return out


def _swiglu(x, perm, top_k, qweight, scales, expert_offsets, x_scale, zero_init, out_dtype, status):
    device = _cabi.one_device(x, perm, qweight, scales, expert_offsets, x_scale, status)
    _check_weight(qweight, scales, 1)
    E, N2, K = qweight.shape
    if N2 % 2:
        raise ValueError("gate and up weights are [E, 2 * I, K]: gate rows, then up rows")
    groups = _groups(expert_offsets, E)
    with _cabi.current_device(device):
        q, sx, out_dtype = _rows(x, x_scale, K, out_dtype)
        code = _out_code(out_dtype)
        T = q.shape[0]
        S = T if perm is None else perm.numel()
        if S and not T:
            raise ValueError("perm lists rows of an empty x")
        h = torch.empty(S, N2 // 2, dtype=out_dtype, device=device)
        qweight, scales = qweight.contiguous(), scales.contiguous()
        offsets = _prepare(expert_offsets, S, groups, N2 // 2, h if zero_init else None, code)
        rc = _cabi.load().mq_w8a8_grouped_swiglu(q.data_ptr(), sx.data_ptr(), _cabi.ptr(perm), T, top_k, qweight.data_ptr(),
                                                 scales.data_ptr(), offsets.data_ptr(), S, groups, E, N2 // 2, K, code,
                                                 h.data_ptr(), _cabi.ptr(status), _cabi.stream_ptr(device))
    _cabi.check(rc, "mq_w8a8_grouped_swiglu")
    _cabi.count_launches(1 if S else 0)
    return h


def w8a8_grouped_swiglu(x: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor, expert_offsets: torch.Tensor,
                        x_scale: torch.Tensor | None = None, zero_init: bool = True, out_dtype: torch.dtype | None = None,
                        status: torch.Tensor | None = None) -> torch.Tensor:
    """``silu(g) * u`` of each expert's rows, g and u the unrounded products with the gate and the up rows of ``qweight``
    (int8 [E, 2I, K]: gate rows first; scales fp32 [E, 2I]); rounded once.  Arguments as in :func:`w8a8_grouped_gemm`."""
    return _swiglu(x, None, 1, qweight, scales, expert_offsets, x_scale, zero_init, out_dtype, status)


def w8a8_grouped_swiglu_gather(x: torch.Tensor, perm: torch.Tensor, top_k: int, qweight: torch.Tensor, scales: torch.Tensor,
                               expert_offsets: torch.Tensor, x_scale: torch.Tensor | None = None,
                               out_dtype: torch.dtype | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`w8a8_grouped_swiglu` on ``x[perm // top_k]`` without materialising the permuted rows: x is the unpermuted [T, K]
    and is quantised once per token.  The result has one row per entry of ``perm`` (int32); rows that no group covers are
    unwritten."""
    if perm.dtype != torch.int32 or perm.dim() != 1 or not perm.is_contiguous():
        raise ValueError("perm is a contiguous int32 vector")
    if top_k < 1:
        raise ValueError("top_k must be positive")
    return _swiglu(x, perm, top_k, qweight, scales, expert_offsets, x_scale, False, out_dtype, status)
