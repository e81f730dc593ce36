"""A long cache's pages that are worth reading: bounds of each page's keys (``page_bounds``) and the choice of pages for a decoded token
by what no key of a page exceeds (``select_pages``), whose tables ``paged_attention`` takes."""
from __future__ import annotations

import torch

from . import _lib, ops
from ._lib import GqkPages, _fast, check, lib
from .attention import _PAGE_TYPES, _TYPES, _heads_view, _strides
from .eager import direct as _direct, stream as _stream, unwatched as _unwatched


def _bounds_into(k_pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, bounds: torch.Tensor, count: int) -> None:
    if lengths.shape[0] == 0 or k_pages.numel() == 0:
        return
    device = k_pages.device
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _bounds_into(k_pages, block_table, lengths, bounds, count)
    n, page, heads, dim = k_pages.shape
    ks = [0 if m == 1 else st for m, st in zip(k_pages.shape, k_pages.stride())]
    pages = GqkPages(k_pages.data_ptr(), None, ks[0], ks[1], ks[2], 0, 0, 0, None, None, _PAGE_TYPES[k_pages.dtype], n, page, heads, dim)
    check(lib.gqk_page_bounds(_lib.byref(pages), block_table.data_ptr(), block_table.stride(0), block_table.shape[1], lengths.data_ptr(),
                              lengths.shape[0], count, bounds.data_ptr(), _stream(device)), "page_bounds")


@torch.library.custom_op("gguf_hip::page_bounds", mutates_args=("bounds",))
def _bounds_op(k_pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, bounds: torch.Tensor, count: int) -> None:
    _bounds_into(k_pages, block_table, lengths, bounds, count)


@_bounds_op.register_fake
def _(k_pages, block_table, lengths, bounds, count):
    return None


def _check_table(what: str, block_table: torch.Tensor, lengths: torch.Tensor, device: torch.device) -> int:
    if lengths.dtype != torch.int32 or lengths.dim() != 1 or lengths.device != device or not lengths.is_contiguous():
        raise ValueError(f"{what}: lengths is contiguous int32 [batch] on {device}")
    batch = lengths.shape[0]
    if (block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != batch or block_table.device != device
            or (block_table.shape[1] > 1 and block_table.stride(1) != 1)):
        raise ValueError(f"{what}: block_table is int32 [{batch}, pages] on {device}, its columns side by side")
    if batch > 65535:
        raise ValueError(f"{what}: {batch} sequences, at most 65535")
    return batch


def page_bounds(k_pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, bounds: torch.Tensor, *,
                count: int = 1) -> torch.Tensor:
    """Brings ``bounds`` up to date for the pages that hold each sequence's last ``count`` keys (the step's new ones): bounds[p, 0] and
    bounds[p, 1] [heads, dim] are the smallest and the largest of page p's keys of that sequence, exactly (NaN where one is).  k_pages [pages, page_size,
    heads, dim] (bf16, fp16 or float8_e4m3fn, strides that are multiples of 8), bounds [pages, 2, heads, dim] of its type, contiguous; block_table int32 [batch, pages] and
    lengths int32 [batch] as paged_attention's.  Keys that were taken back are forgotten, as a page is read anew.  A page that
    several sequences hold must hold the same keys of each.  ``copy_pages`` on bounds follows a fork or a compaction.  Returns bounds."""
    what = "page_bounds"
    if _fast is not None and _unwatched() and _fast.page_bounds(k_pages, block_table, lengths, bounds, count):
        return bounds
    ops._require_gpu(k_pages, what)
    if k_pages.dim() != 4 or k_pages.dtype not in _PAGE_TYPES or k_pages.stride(3) != 1:
        raise ValueError(f"{what}: pages are [pages, page_size, heads, dim], a key's dims side by side, got {k_pages.dtype} "
                         f"{tuple(k_pages.shape)} {k_pages.stride()}")
    n, _, heads, dim = k_pages.shape
    if (bounds.shape != (n, 2, heads, dim) or bounds.dtype != k_pages.dtype or bounds.device != k_pages.device
            or not bounds.is_contiguous()):
        raise ValueError(f"{what}: bounds is contiguous {k_pages.dtype} [{n}, 2, {heads}, {dim}] on {k_pages.device}, got {bounds.dtype} "
                         f"{tuple(bounds.shape)} on {bounds.device}")
    _check_table(what, block_table, lengths, k_pages.device)
    count = int(count)
    if not 0 <= count < 1 << 31:
        raise ValueError(f"{what}: the last {count} keys")
    if _direct(k_pages, block_table, lengths, bounds):
        _bounds_into(k_pages, block_table, lengths, bounds, count)
        torch.autograd.graph.increment_version(bounds)
    else:
        _bounds_op(k_pages, block_table, lengths, bounds, count)
    return bounds


def _select_into(q: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, keep: int, page_size: int, sink: int,
                 recent: int, max_length: int, table: torch.Tensor, kept: torch.Tensor, workspace: torch.Tensor | None) -> None:
    batch, heads, dim = q.shape
    if batch == 0:
        return
    device = q.device
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _select_into(q, bounds, block_table, lengths, keep, page_size, sink, recent, max_length, table, kept, workspace)
    ws = ops.shared_workspace(device) if workspace is None else workspace
    qs = _strides(q)
    check(lib.gqk_select_pages(q.data_ptr(), qs[0], qs[1], _TYPES[q.dtype], batch, heads, bounds.data_ptr(), _PAGE_TYPES[bounds.dtype],
                               bounds.shape[0], bounds.shape[2], dim, block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
                               lengths.data_ptr(), max_length, page_size, keep, sink, recent, table.data_ptr(), kept.data_ptr(),
                               ws.data_ptr(), ws.numel() * ws.element_size(), _stream(device)), "select_pages")


@torch.library.custom_op("gguf_hip::select_pages", mutates_args=("table", "kept", "workspace"))
def _select_op(q: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, keep: int, page_size: int, sink: int,
               recent: int, max_length: int, table: torch.Tensor, kept: torch.Tensor, workspace: torch.Tensor | None) -> None:
    _select_into(q, bounds, block_table, lengths, keep, page_size, sink, recent, max_length, table, kept, workspace)


@_select_op.register_fake
def _(q, bounds, block_table, lengths, keep, page_size, sink, recent, max_length, table, kept, workspace):
    return None


def select_pages(q: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, keep: int, page_size: int, *,
                 sink: int = 1, recent: int = 1, max_length: int | None = None, workspace: torch.Tensor | None = None
                 ) -> tuple[torch.Tensor, torch.Tensor]:
    """The ``keep`` pages of each sequence that its new token attends to, for each key head: the first ``sink``, the last ``recent`` (one
    at least), and of the others those with the largest bound on a key's product with a query of the head's group,
    max over the group of sum_d max(q_d lo_d, q_d hi_d), among equals the first.  q [batch, query heads, dim] (bf16 or fp16); bounds [pages, 2,
    heads, dim] as ``page_bounds`` keeps them (of q's type or float8_e4m3fn: positive scales do not change the order); block_table int32 [batch, pages]
    and lengths int32 [batch] as paged_attention's, ``max_length`` an upper bound on lengths.  Scores are summed in 64 bits, as near equals decide what is
    read.

    Returns (table int32 [batch, heads, keep], lengths int32 [batch]) for ``paged_attention``: the pages in their sequence's order, -1 behind them,
    and the number of keys in them.  A sequence of up to ``keep`` pages keeps all.  A page outside of the cache is taken, and a length
    above max_length becomes 2 ** 31 - 1, so that the attention answers NaN.  ``workspace``: as mul_mat_grouped's (one that does not hold
    the scores of all sequences takes them in turns)."""
    what = "select_pages"
    if _fast is not None and _unwatched():
        got = _fast.select_pages(q, bounds, block_table, lengths, keep, page_size, sink, recent, max_length, workspace)
        if got is not None:
            return got
    ops._require_gpu(q, what)
    if q.dtype not in _TYPES:
        raise ValueError(f"{what}: q is bf16 or fp16, not {q.dtype}")
    q = _heads_view(q, what)
    batch, heads, dim = q.shape
    if (bounds.dim() != 4 or bounds.shape[1] != 2 or bounds.shape[0] < 1 or bounds.shape[3] != dim or bounds.dtype not in (q.dtype, torch.float8_e4m3fn)
            or bounds.device != q.device or not bounds.is_contiguous()):
        raise ValueError(f"{what}: bounds is contiguous [pages, 2, heads, {dim}] of {q.dtype} or float8_e4m3fn on {q.device}, got "
                         f"{bounds.dtype} {tuple(bounds.shape)} on {bounds.device}")
    if heads == 0 or bounds.shape[2] == 0 or heads % bounds.shape[2]:
        raise ValueError(f"{what}: {heads} query heads over {bounds.shape[2]}")
    if _check_table(what, block_table, lengths, q.device) != batch:
        raise ValueError(f"{what}: lengths of {lengths.shape[0]} sequences for {batch}")
    keep, page_size, sink, recent = int(keep), int(page_size), int(sink), int(recent)
    if not 1 <= keep < 1 << 31 or not 1 <= page_size < 1 << 31 or sink < 0 or recent < 1 or sink + recent > keep:
        raise ValueError(f"{what}: {keep} pages of {page_size} tokens, the first {sink} and the last {recent} (one at least) among them")
    ops.check_workspace(workspace, q.device, what)
    room = min(block_table.shape[1] * page_size, _lib.GQK_MAX_KEYS)
    max_length = room if max_length is None else int(max_length)
    if not 0 <= max_length <= room:
        raise ValueError(f"{what}: max_length {max_length} (the table holds {room} keys)")
    table = torch.empty((batch, bounds.shape[2], keep), dtype=torch.int32, device=q.device)
    kept = torch.empty((batch,), dtype=torch.int32, device=q.device)
    args = (q, bounds, block_table, lengths, keep, page_size, sink, recent, max_length, table, kept, workspace)
    if _direct(q, bounds, block_table, lengths, workspace):
        _select_into(*args)
    else:
        _select_op(*args)
    return table, kept
