"""A step of several new tokens per sequence: its tables, slots, positions and masks, built on the GPU from the sequences' lengths
(``step_tables``), so that a captured step serves any mixture of drafted trees, chains and chunks of prompts of the same size."""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib, ops
from ._lib import _fast, check, lib
from .eager import direct as _direct, stream as _stream, unwatched as _unwatched


class StepTables(NamedTuple):
    block_table: torch.Tensor     # int32 [batch, width]: each sequence's pages, -1 behind its last
    lengths: torch.Tensor         # int32 [batch]: keys with the new tokens'
    starts: torch.Tensor          # int32 [batch + 1]: each sequence's rows
    sequences: torch.Tensor       # int32 [tokens]: each row's sequence, -1 behind the last
    positions: torch.Tensor       # int32 [tokens]
    slots: torch.Tensor           # int64 [tokens]: -1 behind the last
    mask: torch.Tensor | None     # int32 [tokens, words]: a drafted token's ancestors and itself


def _tables_into(page_lists: torch.Tensor, requests: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor, parents: torch.Tensor | None,
                 tokens: int, page_size: int, tree: int, block_table: torch.Tensor, totals: torch.Tensor, starts: torch.Tensor,
                 sequences: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, mask: torch.Tensor | None) -> None:
    device = page_lists.device
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _tables_into(page_lists, requests, lengths, counts, parents, tokens, page_size, tree, block_table, totals, starts,
                                sequences, positions, slots, mask)
    n, width = page_lists.shape
    check(lib.gqk_step_tables(page_lists.data_ptr(), page_lists.stride(0) if n > 1 else width, n, width, requests.data_ptr(),
                              requests.dtype == torch.int64, lengths.data_ptr(), counts.data_ptr(), requests.shape[0], tokens, page_size,
                              None if parents is None else parents.data_ptr(), tree, block_table.data_ptr(), totals.data_ptr(),
                              starts.data_ptr(), sequences.data_ptr(), positions.data_ptr(), slots.data_ptr(),
                              None if mask is None else mask.data_ptr(), _stream(device)), "step_tables")


@torch.library.custom_op("gguf_hip::step_tables", mutates_args=("block_table", "totals", "starts", "sequences", "positions", "slots", "mask"))
def _tables_op(page_lists: torch.Tensor, requests: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor, parents: torch.Tensor | None,
               tokens: int, page_size: int, tree: int, block_table: torch.Tensor, totals: torch.Tensor, starts: torch.Tensor,
               sequences: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, mask: torch.Tensor | None) -> None:
    _tables_into(page_lists, requests, lengths, counts, parents, tokens, page_size, tree, block_table, totals, starts, sequences, positions,
                 slots, mask)


@_tables_op.register_fake
def _(page_lists, requests, lengths, counts, parents, tokens, page_size, tree, block_table, totals, starts, sequences, positions, slots, mask):
    return None


def step_tables(page_lists: torch.Tensor, requests: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor, tokens: int, page_size: int,
                *, parents: torch.Tensor | None = None, tree: int = 0) -> StepTables:
    """What a step of new tokens needs to know of them, in one launch.  Sequence b of the batch is request requests[b] (int32 or int64
    [batch]; negative: no sequence, with no new tokens), whose pages are page_lists[requests[b]] (int32 [requests, width]: the lists that a
    server keeps on the GPU, written as its PagePool gives pages); lengths[b] of its keys are in the cache, and counts[b] new tokens come
    (int32 [batch] each).  ``tokens``: the rows of the step, at least the new tokens' number; the rows behind the last have no
    sequence and no slot.  A drafted tree: ``parents`` int32 [tokens], each new token's parent among its sequence's (by its number there,
    -1: the last token of the cache), which comes before it, and ``tree``, the most new tokens of a sequence (up to 1024).

    Returns StepTables: block_table and lengths for ``tree_attention`` and ``paged_attention``, starts and mask for ``tree_attention``,
    positions (a token's own number behind the cache, or the number of its ancestors) and slots for ``qk_norm_rope``, sequences to look up what
    belongs to a request (its adapter).  A sequence that cannot be (no such request, keys beyond its list, more tokens than there are rows
    or than ``tree``) gets a length of 2 ** 31 - 1, for which attention answers NaN, and no slots; a token whose parent does not come before
    it position -1 and an empty mask, and so do those below it."""
    what = "step_tables"
    if _fast is not None and _unwatched():
        got = _fast.step_tables(page_lists, requests, lengths, counts, tokens, page_size, parents, tree)
        if got is not None:
            return StepTables(*got)
    ops._require_gpu(page_lists, what)
    device = page_lists.device
    if (page_lists.dtype != torch.int32 or page_lists.dim() != 2 or (page_lists.shape[1] > 1 and page_lists.stride(1) != 1)
            or (page_lists.shape[0] > 1 and page_lists.stride(0) < page_lists.shape[1])):
        raise ValueError(f"{what}: page_lists is int32 [requests, pages], its columns side by side, got {page_lists.dtype} "
                         f"{tuple(page_lists.shape)} {page_lists.stride()}")
    if requests.dim() != 1 or requests.dtype not in (torch.int32, torch.int64) or requests.device != device or not requests.is_contiguous():
        raise ValueError(f"{what}: requests is contiguous int32 or int64 [batch] on {device}")
    batch, tokens, page_size, tree = requests.shape[0], int(tokens), int(page_size), int(tree)
    for t in (lengths, counts):
        if t.dtype != torch.int32 or t.shape != (batch,) or t.device != device or not t.is_contiguous():
            raise ValueError(f"{what}: lengths and counts are contiguous int32 [{batch}] on {device}")
    if tokens < 0 or tokens >= 1 << 31 or page_size < 1 or page_size >= 1 << 31 or batch > 65535:
        raise ValueError(f"{what}: {batch} sequences (at most 65535), {tokens} tokens, pages of {page_size}")
    if (parents is None) != (tree == 0) or not 0 <= tree <= _lib.GQK_MAX_TREE:
        raise ValueError(f"{what}: a tree is its parents and the most tokens of one, up to {_lib.GQK_MAX_TREE}; got {tree}")
    if parents is not None and (parents.dtype != torch.int32 or parents.shape != (tokens,) or parents.device != device
                                or not parents.is_contiguous()):
        raise ValueError(f"{what}: parents is contiguous int32 [{tokens}] on {device}")
    i32 = lambda *s: torch.empty(s, dtype=torch.int32, device=device)  # noqa: E731
    got = StepTables(i32(batch, page_lists.shape[1]), i32(batch), i32(batch + 1), i32(tokens), i32(tokens),
                     torch.empty((tokens,), dtype=torch.int64, device=device), i32(tokens, (tree + 31) // 32) if tree else None)
    args = (page_lists, requests, lengths, counts, parents, tokens, page_size, tree, *got)
    if _direct(page_lists, requests, lengths, counts, parents):
        _tables_into(*args)
    else:
        _tables_op(*args)
    return got
