"""Low-rank adapters of many requests beside a shared projection: ``lora_add`` adds to a layer's output
(``mul_mat_grouped``, ``GGUFLinearMethod.apply``) what each row's own adapter contributes.  Two launches on the current
stream (one for a few rows); which rows go with which adapter is found on the GPU from the row's index, so a batch may change between
the replays of a HIP graph."""
from __future__ import annotations

import ctypes
from functools import lru_cache

import torch

from . import _lib, ops
from ._lib import _fast, check, lib
from .eager import direct as _direct, no_backward, stream as _stream, unwatched as _unwatched

_TYPES = {torch.bfloat16: _lib.GQK_DTYPE_BF16, torch.float16: _lib.GQK_DTYPE_F16}
MAX_PARTS, MAX_RANK, MAX_K = 8, 256, (1 << 22) - 8
MAX_ROWS = 65535 * 64   # of one launch


@lru_cache(maxsize=256)
def _columns(n_outs: tuple[int, ...]):
    return (ctypes.c_int64 * len(n_outs))(*n_outs)


def _lora_into(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor,
               scales: torch.Tensor | None, n_outs: tuple[int, ...], out: torch.Tensor, workspace: torch.Tensor | None) -> None:
    M, K = x.shape
    if M == 0:
        return
    device = x.device
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _lora_into(y, x, a, b, ids, scales, n_outs, out, workspace)
    ws = ops.shared_workspace(device) if workspace is None else workspace
    have = ws.numel() * ws.element_size()
    slots, parts, rank, _ = a.shape
    wide, size = ids.dtype == torch.int64, ids.element_size()
    # rows are independent: what does not fit the workspace at once goes in turns (a last, shorter one that would like more room
    # than the others gets fewer splits of K)
    rows = M
    while rows > MAX_ROWS or rows > 1 and check(lib.gqk_lora_workspace_bytes(rows, K, parts, rank), "lora_add") > have:
        rows = (rows + 1) // 2
    ys, xs, os = (t.stride(0) if M > 1 else t.shape[1] for t in (y, x, out))   # of one row alone it means nothing
    for r in range(0, M, rows):
        check(lib.gqk_lora_add(y.data_ptr() + 2 * r * ys, ys, x.data_ptr() + 2 * r * xs, xs, min(rows, M - r), K, a.data_ptr(),
                               b.data_ptr(), slots, parts, _columns(n_outs), rank, ids.data_ptr() + r * size, wide,
                               None if scales is None else scales.data_ptr(), _TYPES[x.dtype], out.data_ptr() + 2 * r * os, os,
                               ws.data_ptr(), have, _stream(device)), "lora_add")


@torch.library.custom_op("gguf_hip::lora_add", mutates_args=("out", "workspace"))
def _lora_op(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor,
             scales: torch.Tensor | None, n_outs: list[int], out: torch.Tensor, workspace: torch.Tensor | None) -> None:
    _lora_into(y, x, a, b, ids, scales, tuple(n_outs), out, workspace)


@_lora_op.register_fake
def _(y, x, a, b, ids, scales, n_outs, out, workspace):
    return None


@torch.library.custom_op("gguf_hip::lora_add_", mutates_args=("y", "workspace"))
def _lora_inplace_op(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor,
                     scales: torch.Tensor | None, n_outs: list[int], workspace: torch.Tensor | None) -> None:
    _lora_into(y, x, a, b, ids, scales, tuple(n_outs), y, workspace)


@_lora_inplace_op.register_fake
def _(y, x, a, b, ids, scales, n_outs, workspace):
    return None


def lora_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor,
             scales: torch.Tensor | None, n_outs, *, out: torch.Tensor | None = None,
             workspace: torch.Tensor | None = None) -> torch.Tensor:
    """y [M, N] plus each row's adapter: row m of x [M, K] with adapter i = ids[m] adds scales[i] * b[i] @ (a[i] @ x[m])
    to the columns of each part.  ``n_outs``: the columns of the parts that the projection merges (q, k, v; gate, up;
    one part: [N]), their sum N; a [adapters, parts, rank, K] and b [adapters, N, rank] as ``pack_adapters`` makes
    them, of x's and y's type (bf16 or fp16), contiguous, K and rank multiples of 8, rank up to 256; scales fp32 [adapters] or None (1); ids
    int32 or int64 [M], negative for a row without an adapter (one beyond the adapters gives a row of NaN).
    Returns a new tensor, or ``out`` (a [M, N] view with unit column stride), which may be y itself, or x.  No backward pass.
    ``workspace``: as mul_mat_grouped's (its own for calls on concurrent streams)."""
    what = "lora_add"
    if _fast is not None and _unwatched():
        got = _fast.lora_add(y, x, a, b, ids, scales, n_outs, out, workspace)
        if got is not None:
            return got
    ops._require_gpu(x, what)
    n_outs = tuple(int(n) for n in n_outs)
    if x.dtype not in _TYPES or x.dim() != 2:
        raise ValueError(f"{what}: x is bf16 or fp16 [rows, K], got {x.dtype} {tuple(x.shape)}")
    M, K = x.shape
    N = sum(n_outs)
    if not n_outs or min(n_outs) < 1 or len(n_outs) > MAX_PARTS:
        raise ValueError(f"{what}: {len(n_outs)} parts (1 to {MAX_PARTS}) of {n_outs} columns")
    if a.dim() != 4 or a.shape[1] != len(n_outs) or a.shape[3] != K or b.shape != (a.shape[0], N, a.shape[2]):
        raise ValueError(f"{what}: a {tuple(a.shape)} is [adapters, {len(n_outs)}, rank, {K}], b {tuple(b.shape)} [adapters, "
                         f"{N}, rank]")
    for t in (a, b):
        if t.dtype != x.dtype or t.device != x.device or not t.is_contiguous() or not ops._addr_aligned(t, 16):
            raise ValueError(f"{what}: a and b are contiguous, 16-byte aligned {x.dtype} on {x.device}")
    if K == 0 or K % 8 or K > MAX_K or a.shape[2] < 8 or a.shape[2] % 8 or a.shape[2] > MAX_RANK:
        raise ValueError(f"{what}: K {K} and rank {a.shape[2]} must be multiples of 8, the rank at most {MAX_RANK}, K {MAX_K}")
    for t in (y, out):
        if t is not None and (t.shape != (M, N) or t.dtype != x.dtype or t.device != x.device):
            raise ValueError(f"{what}: y and out are {x.dtype} [{M}, {N}] on {x.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if ids.dtype not in (torch.int32, torch.int64) or ids.shape != (M,) or ids.device != x.device or not ids.is_contiguous():
        raise ValueError(f"{what}: ids is contiguous int32 or int64 [{M}] on {x.device}")
    if scales is not None and (scales.dtype != torch.float32 or scales.shape != (a.shape[0],) or scales.device != x.device
                               or not scales.is_contiguous()):
        raise ValueError(f"{what}: scales is contiguous fp32 [{a.shape[0]}] on {x.device}")
    ops.check_workspace(workspace, x.device, what)
    if out is not None and out.numel() and ((N > 1 and out.stride(1) != 1) or (M > 1 and out.stride(0) < N)):
        raise ValueError(f"{what}: out's columns must lie side by side, got strides {out.stride()}")
    inplace = out is y
    if (N > 1 and y.stride(1) != 1) or (M > 1 and y.stride(0) < N):
        y = y.contiguous()
    if x.stride(1) != 1 or (M > 1 and (x.stride(0) % 8 or not K <= x.stride(0) <= MAX_K)) or not ops._addr_aligned(x, 16):
        x = x.clone(memory_format=torch.contiguous_format)
    if out is None:
        out = torch.empty((M, N), dtype=x.dtype, device=x.device)
    if _direct(y, x, a, b, ids, scales, out, workspace):
        _lora_into(y, x, a, b, ids, scales, n_outs, out, workspace)
        torch.autograd.graph.increment_version(out)
    elif inplace:
        _lora_inplace_op(out, x, a, b, ids, scales, list(n_outs), workspace)
    else:
        _lora_op(y, x, a, b, ids, scales, list(n_outs), out, workspace)
    no_backward(what, out, y, x, a, b, scales)
    return out


def pack_adapters(adapters, n_outs, K: int, dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda",
                  rank: int | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(a, b, scales) of a projection for ``lora_add``: ``adapters`` is a list with, for each slot, None or
    (A parts, B parts, scale), a part's A [r, K] and B [columns, r] being None where the adapter leaves it alone.  Ranks
    may differ: all are padded with zeros to ``rank`` (default: the largest, rounded up to a multiple of 8)."""
    n_outs = [int(n) for n in n_outs]
    most = max([A.shape[0] for ad in adapters if ad is not None for A in ad[0] if A is not None], default=8)
    rank = (most + 7) // 8 * 8 if rank is None else int(rank)
    if rank < most or rank % 8 or rank > MAX_RANK or rank < 8:
        raise ValueError(f"pack_adapters: rank {rank} for adapters of up to {most} (a multiple of 8, at most {MAX_RANK})")
    a = torch.zeros((len(adapters), len(n_outs), rank, K), dtype=dtype, device=device)
    b = torch.zeros((len(adapters), sum(n_outs), rank), dtype=dtype, device=device)
    scales = torch.zeros(len(adapters), dtype=torch.float32, device=device)
    for i, ad in enumerate(adapters):
        if ad is None:
            continue
        As, Bs, scale = ad
        if len(As) != len(n_outs) or len(Bs) != len(n_outs):
            raise ValueError(f"pack_adapters: adapter {i} has {len(As)} / {len(Bs)} parts of {len(n_outs)}")
        scales[i] = float(scale)
        col = 0
        for p, (A, B, n) in enumerate(zip(As, Bs, n_outs)):
            if (A is None) != (B is None) or (A is not None and (A.dim() != 2 or A.shape[1] != K or B.shape != (n, A.shape[0]))):
                raise ValueError(f"pack_adapters: adapter {i}, part {p}: A is [r, {K}] and B [{n}, r], or both None")
            if A is not None:
                a[i, p, :A.shape[0]] = A
                b[i, col:col + n, :A.shape[0]] = B
            col += n
    return a, b, scales
