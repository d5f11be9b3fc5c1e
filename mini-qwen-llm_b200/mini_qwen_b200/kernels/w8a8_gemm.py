"""W8A8 products: int8 weights with a scale for each output channel, int8 activations with a scale for each token.

The reference has no 8-bit path; the calls stand beside :mod:`.w4a16_gemm` and :mod:`.moe_grouped_gemm` and follow their shapes.
Activations are given as bf16, fp16 or fp32 rows, which the call quantises itself, or as int8 rows together with their scales
(``x_scale``, from :func:`quantize_rows_int8`) where several products read the same rows."""
from __future__ import annotations

import ctypes
import functools
import threading

import torch

from .. import _cabi

MAX_K = 131071      # 128 * 128 * K < 2^31: the int32 sums are exact


class _Launches(threading.local):
    """Where a call of this host thread says how many kernels it launched."""

    def __init__(self):
        self.word = ctypes.c_int32(0)
        self.address = ctypes.addressof(self.word)


_launches = _Launches()


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(rows: int, K: int, groups: int) -> int:
    return _cabi.load().mq_w8a8_workspace_bytes(rows, K, groups)


def _apart(x: torch.Tensor, K: int) -> torch.Tensor:
    """x as rows of K that may lie apart but are dense in themselves."""
    rows = x if x.dim() == 2 else x.reshape(-1, K)
    if rows.stride(1) != 1 and K > 1 or rows.stride(0) < 0:
        rows = rows.contiguous()
    return rows


def quantize_rows_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., K] -> (q int8 [..., K] in -127..127, scale fp32 [...]): ``scale = max|row| / 127`` rounded to fp32 and
    ``q = round(row / scale)``, halves to even.  A row of zeros has scale 0; a row that holds an infinity or a NaN has scale NaN
    and q 0, so that what is computed from it is NaN.  Rows may lie apart (a slice of wider rows is read in place)."""
    index = _cabi.one_device(x)
    shape = x.shape
    if not shape or shape[-1] == 0:
        raise ValueError("rows to quantise are [..., K] with K >= 1")
    code = _cabi.dtype_code(x)
    K = shape[-1]
    rows = _apart(x, K)
    q = torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format)
    scale = x.new_empty(shape[:-1], dtype=torch.float32)
    T = rows.shape[0]
    rc = _cabi.on_device(index, _cabi.load().mq_quantize_rows_int8, rows.data_ptr(), code, T, K, rows.stride(0), q.data_ptr(),
                         scale.data_ptr(), _cabi.stream_ptr(index))
    if rc:
        _cabi.check(rc, "mq_quantize_rows_int8")
    _cabi.count_launches(1 if T else 0)
    return q, scale


def _check_weight(qweight, scales, lead: int):
    if qweight.dtype != torch.int8 or scales.dtype != torch.float32:
        raise ValueError("weights are int8 with float32 scales")
    shape = qweight.shape
    if len(shape) != lead + 2 or scales.shape != shape[:-1]:
        raise ValueError(f"weights are {'[E, N, K]' if lead else '[N, K]'} with a scale for each output channel; got "
                         f"{tuple(shape)} and {tuple(scales.shape)}")
    if not 1 <= shape[-1] <= MAX_K:
        raise ValueError(f"K must be 1..{MAX_K}, got {shape[-1]}")
    if 0 in shape:
        raise ValueError("the weights have no output channels")


def _rows(x, x_scale, K, out_dtype):
    """(the rows, their scales, their type's code or None for int8, the type of the result and its code)."""
    if x.dim() != 2 or x.shape[1] != K:
        raise ValueError(f"activations are [rows, {K}], got {tuple(x.shape)}")
    if x.dtype == torch.int8:
        if x_scale is None or x_scale.dtype != torch.float32 or x_scale.shape != x.shape[:1]:
            raise ValueError("int8 activations come with x_scale, float32 [rows]")
        x, x_scale, code = x.contiguous(), x_scale.contiguous(), None
        out_dtype = torch.bfloat16 if out_dtype is None else out_dtype
    else:
        if x_scale is not None:
            raise ValueError("x_scale belongs to int8 activations")
        x, code = _apart(x, K), _cabi.dtype_code(x)
        out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in _cabi._DTYPES:
        raise ValueError(f"unsupported result dtype {out_dtype}; expected float32, bfloat16 or float16")
    return x, x_scale, code, out_dtype, _cabi._DTYPES[out_dtype]


def w8a8_gemm(x: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor, x_scale: torch.Tensor | None = None,
              out_dtype: torch.dtype | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """``(q @ qweight.T) * x_scale[:, None] * scales`` with q and x_scale the int8 rows of x; [M, N].

    x [M, K] bf16, fp16 or fp32, or int8 with ``x_scale`` [M]; qweight int8 [N, K]; scales fp32 [N].  The result has x's type
    (bf16 for int8 rows) unless ``out_dtype`` says otherwise.  ``status`` (int32 [1], optional) receives device-side error bits
    (a bounded wait that ran out)."""
    index = _cabi.one_device(x, qweight, scales, x_scale, status)
    _check_weight(qweight, scales, 0)
    N, K = qweight.shape
    x, x_scale, code, out_dtype, out_code = _rows(x, x_scale, K, out_dtype)
    if not (qweight.is_contiguous() and scales.is_contiguous()):
        qweight, scales = qweight.contiguous(), scales.contiguous()
    M = x.shape[0]
    lib, stream = _cabi.load(), _cabi.stream_ptr(index)
    out = x.new_empty((M, N), dtype=out_dtype)
    word = None if status is None else status.data_ptr()
    if code is None:
        rc = _cabi.on_device(index, lib.mq_w8a8_linear, x.data_ptr(), x_scale.data_ptr(), qweight.data_ptr(), scales.data_ptr(),
                             M, N, K, out_code, out.data_ptr(), word, stream)
        launched = 1 if M else 0
    else:
        space, ws = 0, None
        # a few rows of few enough channels are quantised and multiplied in one launch, without a workspace
        if M > 16 or M * K > 16384 or N > 4096 or K % 16 or x.data_ptr() % 16 or qweight.data_ptr() % 16 or x.stride(0) % 8:
            space = _workspace_bytes(M, K, 0)
            ws = x.new_empty(space, dtype=torch.uint8)
        rc = _cabi.on_device(index, lib.mq_w8a8_linear_x, x.data_ptr(), code, x.stride(0), qweight.data_ptr(), scales.data_ptr(),
                             M, N, K, out_code, None if ws is None else ws.data_ptr(), space, out.data_ptr(), word,
                             _launches.address, stream)
        launched = _launches.word.value
    if rc:
        _cabi.check(rc, "mq_w8a8_linear")
    _cabi.count_launches(launched)
    return out


def _groups(expert_offsets, E: int) -> int:
    if expert_offsets.dim() != 1 or expert_offsets.dtype not in (torch.int32, torch.int64):
        raise ValueError("expert_offsets are one-dimensional int32 or int64")
    groups = expert_offsets.numel() - 1
    if groups < E or groups % E:
        raise ValueError(f"expert_offsets hold {groups} groups; the weights hold {E} experts")
    return groups


def _grouped(what, x, perm, top_k, qweight, scales, expert_offsets, x_scale, zero_init, out, out_dtype, status):
    """Both grouped products: plain, or gate and up with SwiGLU."""
    index = _cabi.one_device(x, perm, qweight, scales, expert_offsets, x_scale, out, status)
    swiglu = what == "mq_w8a8_grouped_swiglu"
    _check_weight(qweight, scales, 1)
    E, N, K = qweight.shape
    if swiglu:
        if N % 2:
            raise ValueError("gate and up weights are [E, 2 * I, K]: gate rows, then up rows")
        N //= 2
    groups = _groups(expert_offsets, E)
    if out is not None:
        if out_dtype is not None and out.dtype != out_dtype:
            raise ValueError("out and out_dtype differ")
        out_dtype = out.dtype
        if tuple(out.shape) != (x.shape[0], N) or not out.is_contiguous():
            raise ValueError(f"out must be contiguous [{x.shape[0]}, {N}]")
    x, x_scale, code, out_dtype, out_code = _rows(x, x_scale, K, out_dtype)
    T = x.shape[0]
    S = T if perm is None else perm.numel()
    if S and not T:
        raise ValueError("perm lists rows of an empty x")
    zero = out is None and zero_init
    if out is None:
        out = x.new_empty((S, N), dtype=out_dtype)
    if not (qweight.is_contiguous() and scales.is_contiguous() and expert_offsets.is_contiguous()):
        qweight, scales, expert_offsets = qweight.contiguous(), scales.contiguous(), expert_offsets.contiguous()
    wide = expert_offsets.dtype == torch.int64
    lib, stream = _cabi.load(), _cabi.stream_ptr(index)
    if code is None:
        launched = 1 if S else 0
        off = expert_offsets
        if S and (zero or wide):
            narrow = x.new_empty(groups + 1, dtype=torch.int32) if wide else None
            rc = _cabi.on_device(index, lib.mq_grouped_prepare, off.data_ptr(), int(wide), S, groups, N, out_code,
                                 out.data_ptr() if zero else None, _cabi.ptr(narrow), None, stream)
            _cabi.check(rc, "mq_grouped_prepare")
            off, launched = narrow if wide else off, 2
        args = (off.data_ptr(), S, groups, E, N, K, out_code, out.data_ptr(), _cabi.ptr(status), stream)
        if swiglu:
            rc = _cabi.on_device(index, lib.mq_w8a8_grouped_swiglu, x.data_ptr(), x_scale.data_ptr(), _cabi.ptr(perm), T, top_k,
                                 qweight.data_ptr(), scales.data_ptr(), *args)
        else:
            rc = _cabi.on_device(index, lib.mq_w8a8_grouped_gemm, x.data_ptr(), x_scale.data_ptr(), qweight.data_ptr(),
                                 scales.data_ptr(), *args)
    else:
        space = _workspace_bytes(T, K, groups)
        ws = x.new_empty(space, dtype=torch.uint8)
        rc = _cabi.on_device(index, lib.mq_w8a8_grouped_x, x.data_ptr(), code, x.stride(0), _cabi.ptr(perm), T, top_k,
                             qweight.data_ptr(), scales.data_ptr(), expert_offsets.data_ptr(), int(wide), S, groups, E, N, K,
                             int(swiglu), int(zero), out_code, ws.data_ptr(), space, out.data_ptr(), _cabi.ptr(status),
                             _launches.address, stream)
        launched = _launches.word.value
    if rc:
        _cabi.check(rc, what)
    _cabi.count_launches(launched)
    return out


def w8a8_grouped_gemm(x: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor, expert_offsets: torch.Tensor,
                      x_scale: torch.Tensor | None = None, zero_init: bool = True, out: torch.Tensor | None = None,
                      out_dtype: torch.dtype | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`w8a8_gemm` of rows ``offsets[e]:offsets[e+1]`` with the weight of expert e.

    qweight int8 [E, N, K], scales fp32 [E, N], offsets [E+1] ascending (or G * E groups, group g on expert g % E).  Rows that no
    group covers are zero (``zero_init=False``: unwritten); with ``out`` given they keep what they hold."""
    return _grouped("mq_w8a8_grouped_gemm", x, None, 1, qweight, scales, expert_offsets, x_scale, zero_init, out, out_dtype,
                    status)


def w8a8_grouped_swiglu(x: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor, expert_offsets: torch.Tensor,
                        x_scale: torch.Tensor | None = None, zero_init: bool = True, out_dtype: torch.dtype | None = None,
                        status: torch.Tensor | None = None) -> torch.Tensor:
    """``silu(g) * u`` of each expert's rows, g and u the unrounded products with the gate and the up rows of ``qweight``
    (int8 [E, 2I, K]: gate rows first; scales fp32 [E, 2I]); rounded once.  Arguments as in :func:`w8a8_grouped_gemm`."""
    return _grouped("mq_w8a8_grouped_swiglu", x, None, 1, qweight, scales, expert_offsets, x_scale, zero_init, None, out_dtype,
                    status)


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
    return _grouped("mq_w8a8_grouped_swiglu", x, perm, top_k, qweight, scales, expert_offsets, x_scale, False, None, out_dtype,
                    status)
