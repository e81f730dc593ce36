"""Between a layer's projections: the residual's addition and the RMS norm of whole rows in one pass (``add_rms_norm``), or with the
result in 8 bits and its scales (``add_rms_norm_fp8``).  One launch on the current stream; only the outputs are allocated; under tracing
one custom op with a fake."""
from __future__ import annotations

import torch

from . import _lib, ops
from ._lib import _fast, check, lib
from .eager import direct as _direct, no_backward, stream as _stream, unwatched as _unwatched

_TYPES = {torch.bfloat16: _lib.GQK_DTYPE_BF16, torch.float16: _lib.GQK_DTYPE_F16}
F8 = torch.float8_e4m3fn


def _row(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _rows(t: torch.Tensor) -> bool:
    """Whether t is rows as the kernel reads them: columns side by side, rows that do not overlap."""
    return (t.shape[1] <= 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1])


def _shared(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.untyped_storage()._cdata == b.untyped_storage()._cdata


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether rows as above, of any two types, have bytes in common."""
    n, own, other = a.shape[0], a.shape[1] * a.element_size(), b.shape[1] * b.element_size()
    row, far = _row(a) * a.element_size(), _row(b) * b.element_size()
    at, to = a.storage_offset() * a.element_size(), b.storage_offset() * b.element_size()
    if not _shared(a, b) or at + (n - 1) * row + own <= to or to + (b.shape[0] - 1) * far + other <= at:
        return False
    return n == 1 or row != far or not own <= (to - at) % row <= row - other   # (columns of one tensor lie between each other's rows)


def _meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of one type and shape, rows as above, share memory otherwise than row by row the same."""
    return (a.storage_offset(), _row(a)) != (b.storage_offset(), _row(b)) and _overlap(a, b)


def _norm_into(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor | None, eps: float, flags: int, group: int,
               out: torch.Tensor, scale: torch.Tensor | None, out_residual: torch.Tensor | None) -> None:
    rows, dim = x.shape
    if rows == 0:
        return
    device = x.device
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _norm_into(x, residual, weight, eps, flags, group, out, scale, out_residual)
    dtype = _TYPES[x.dtype]
    check(lib.gqk_add_rms_norm(x.data_ptr(), _row(x), None if residual is None else residual.data_ptr(),
                               0 if residual is None else _row(residual), dtype, rows, dim, None if weight is None else weight.data_ptr(),
                               dtype if weight is None or weight.dtype == x.dtype else _lib.GQK_DTYPE_F32, eps, flags, out.data_ptr(),
                               _row(out), _lib.GQK_DTYPE_FP8 if out.dtype == F8 else dtype, None if scale is None else scale.data_ptr(),
                               group, None if out_residual is None else out_residual.data_ptr(),
                               0 if out_residual is None else _row(out_residual), _stream(device)), "add_rms_norm")


@torch.library.custom_op("gguf_hip::add_rms_norm", mutates_args=("out", "scale", "out_residual"))
def _norm_op(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor | None, eps: float, flags: int, group: int,
             out: torch.Tensor, scale: torch.Tensor | None, out_residual: torch.Tensor | None) -> None:
    _norm_into(x, residual, weight, eps, flags, group, out, scale, out_residual)


@_norm_op.register_fake
def _(x, residual, weight, eps, flags, group, out, scale, out_residual):
    return None


def _call(what: str, x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor | None, eps: float, unit_offset: bool, f8: bool,
          group: int, out: torch.Tensor | None, out_residual: torch.Tensor | None):
    flags = _lib.GQK_ROPE_UNIT_OFFSET if unit_offset else 0
    if _fast is not None and _unwatched():
        got = _fast.add_rms_norm(x, residual, weight, eps, flags, f8, group, out, out_residual)
        if got is not None:
            return got
    ops._require_gpu(x, what)
    if x.dtype not in _TYPES or x.dim() != 2 or not 1 <= x.shape[1] <= _lib.GQK_NORM_MAX_DIM:
        raise ValueError(f"{what}: x is bf16 or fp16 [rows, dim (1 to {_lib.GQK_NORM_MAX_DIM})], got {x.dtype} {tuple(x.shape)}")
    rows, dim = x.shape
    for t in (residual, out_residual, None if f8 else out):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype or t.device != x.device):
            raise ValueError(f"{what}: the residual and the outputs are {x.dtype} [{rows}, {dim}] on {x.device}, got {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")
    if f8 and out is not None and (out.shape != x.shape or out.dtype != F8 or out.device != x.device):
        raise ValueError(f"{what}: out is {F8} [{rows}, {dim}] on {x.device}, got {out.dtype} {tuple(out.shape)} on {out.device}")
    if out_residual is not None and residual is None:
        raise ValueError(f"{what}: out_residual without a residual")
    if weight is not None and (weight.shape != (dim,) or weight.dtype not in (x.dtype, torch.float32) or weight.device != x.device
                               or not weight.is_contiguous()):
        raise ValueError(f"{what}: weight is contiguous {x.dtype} or fp32 [{dim}] on {x.device}")
    if weight is None and unit_offset:
        raise ValueError(f"{what}: an offset without weights")
    if group and (group not in (32, 64, 128, 256, 512) or dim % group):
        raise ValueError(f"{what}: groups of {group} columns of {dim} (0, or a power of two from 32 to 512 that divides them)")
    for t in (out, out_residual):
        if t is not None and t.numel() and not _rows(t):
            raise ValueError(f"{what}: an output's columns must lie side by side, got strides {t.stride()}")
    if f8 and out is not None and out.numel():
        # (an input that is not rows is copied before)
        if any(t is not None and _rows(t) and _overlap(t, out) for t in (x, residual, None if weight is None else weight[None], out_residual)):
            raise ValueError(f"{what}: out in 8 bits is memory of its own")
    both = [t for t in (out, out_residual) if t is not None and t.numel()]
    if not f8 and len(both) == 2 and ((_shared(*both) and both[0].storage_offset() == both[1].storage_offset()) or _meet(*both)):
        raise ValueError(f"{what}: out and out_residual share memory")
    new_out, new_residual = out is None, residual is not None and out_residual is None
    if new_out:
        out = torch.empty((rows, dim), dtype=F8 if f8 else x.dtype, device=x.device)
    if new_residual:
        out_residual = torch.empty((rows, dim), dtype=x.dtype, device=x.device)
    scale = torch.empty((rows, dim // group if group else 1), dtype=torch.float32, device=x.device) if f8 else None
    # an input that a kernel cannot read as it is, or that shares memory with an output of another layout, is copied
    both = [t for t in both if t.dtype == x.dtype]
    a, b = (t if t is None or t.numel() == 0 or (_rows(t) and not any(_meet(t, o) for o in both)) else
            t.clone(memory_format=torch.contiguous_format) for t in (x, residual))
    if weight is not None and any(_shared(weight, o) for o in both):
        weight = weight.clone()
    args = (a, b, weight, float(eps), flags, int(group), out, scale, out_residual)
    if _direct(x, residual, weight, out, out_residual):
        _norm_into(*args)
        for t in (out, out_residual):
            if t is not None:
                torch.autograd.graph.increment_version(t)
    else:
        # an op's output is not its input too: in place, it goes to new tensors first
        o = torch.empty_like(out, memory_format=torch.contiguous_format) if not new_out else out
        r = torch.empty_like(out_residual, memory_format=torch.contiguous_format) if out_residual is not None and not new_residual else out_residual
        _norm_op(a, b, weight, float(eps), flags, int(group), o, scale, r)
        with torch.no_grad():
            if o is not out:
                out.copy_(o)
            if r is not out_residual:
                out_residual.copy_(r)
    no_backward(what, out, x, residual, weight)
    no_backward(what, out_residual, x, residual)
    no_backward(what, scale, x, residual, weight)
    return (out, scale, out_residual) if f8 else (out, out_residual)


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor | None = None, *, eps: float = 1e-6,
                 unit_offset: bool = False, out: torch.Tensor | None = None, out_residual: torch.Tensor | None = None):
    """s = x + residual and its RMS norm, s rsqrt(mean(s ** 2) + eps) * weight, of rows x [rows, dim] (bf16 or fp16, any strides between rows,
    dim up to 32768).  ``weight`` [dim] of x's type or fp32 (``unit_offset``: 1 + weight; None: no weight); residual None: of x alone.  Sums are
    in 32 bits, the norm is of s before it is rounded.  Returns (normed rows, s), s None without a residual: new tensors, or ``out`` /
    ``out_residual``, which may be x or residual themselves, but share no memory with each other.  No backward pass."""
    return _call("add_rms_norm", x, residual, weight, eps, unit_offset, False, 0, out, out_residual)


def add_rms_norm_fp8(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor | None = None, *, eps: float = 1e-6,
                     unit_offset: bool = False, group: int = 0, out: torch.Tensor | None = None,
                     out_residual: torch.Tensor | None = None):
    """``add_rms_norm`` with the normed rows in float8_e4m3fn and their scales: (values, scales, s), values * scales being the rows.
    Scales are fp32 [rows, 1], or [rows, dim / group] for each ``group`` columns (a power of two from 32 to 512 that divides dim): the largest
    size of a value (2 ** -100 at least) / 448.  ``out``: float8_e4m3fn [rows, dim], bytes of its own.  No backward pass."""
    return _call("add_rms_norm_fp8", x, residual, weight, eps, unit_offset, True, group, out, out_residual)
