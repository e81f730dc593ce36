"""The pages of a key-value cache: which are free, shared or a sequence's own (``PagePool``, on the host), and the
copies between them on the GPU (``copy_pages``, one launch for each 448 pairs, of all layers)."""
from __future__ import annotations

import heapq

import numpy as np
import torch

from . import ops
from ._lib import _fast, check, lib
from .eager import direct as _direct, stream as _stream, unwatched as _unwatched


def _pairs(t, what: str) -> np.ndarray:
    if isinstance(t, torch.Tensor):
        if t.is_cuda:
            raise ValueError(f"{what}: page numbers are the host's (a list, an array or a CPU tensor)")
        t = t.numpy()
    a = np.asarray(t)
    if a.size == 0:
        return np.empty(0, np.int32)
    if a.ndim != 1 or a.dtype.kind not in "iu":
        raise ValueError(f"{what}: page numbers are a list of integers")
    if a.dtype != np.int32:
        if a.min() < -2 ** 31 or a.max() >= 2 ** 31:
            raise ValueError(f"{what}: page number out of range")
        a = a.astype(np.int32)
    return np.ascontiguousarray(a)


def _layout(pages: torch.Tensor, dim: int) -> tuple[int, int, int, int, int]:
    """(planes, elements from one to the next, pages, elements from one to the next, elements of a page)."""
    what = "copy_pages"
    shape, stride = pages.shape, pages.stride()
    n = 1
    for m, st in zip(reversed(shape[dim + 1:]), reversed(stride[dim + 1:])):
        if m != 1 and st != n:
            raise ValueError(f"{what}: a page's own dimensions must be contiguous, got strides {stride}")
        n *= m
    planes, plane = 1, 0
    for m, st in zip(reversed(shape[:dim]), reversed(stride[:dim])):
        if m == 1:
            continue
        if planes > 1 and st != plane * planes:
            raise ValueError(f"{what}: the dimensions before the pages must be evenly spaced, got strides {stride}")
        plane = st if planes == 1 else plane
        planes *= m
    if pages.numel() == 0:
        planes = 0
    return planes, plane, shape[dim], stride[dim] if shape[dim] > 1 else n, n


def _copy_into(pages: torch.Tensor, src: np.ndarray, dst: np.ndarray, dim: int) -> None:
    if pages.device.index != torch.cuda.current_device():
        with torch.cuda.device(pages.device):
            return _copy_into(pages, src, dst, dim)
    planes, plane, count, page, n = _layout(pages, dim)
    size = pages.element_size()
    check(lib.gqk_copy_pages(pages.data_ptr(), planes, plane * size, count, page * size, n * size, src.ctypes.data, dst.ctypes.data,
                             src.size, _stream(pages.device)), "copy_pages")


@torch.library.custom_op("gguf_hip::copy_pages", mutates_args=("pages",))
def _copy_op(pages: torch.Tensor, src: list[int], dst: list[int], dim: int) -> None:
    _copy_into(pages, np.array(src, np.int32), np.array(dst, np.int32), dim)


@_copy_op.register_fake
def _(pages, src, dst, dim):
    return None


def copy_pages(pages: torch.Tensor, src, dst, dim: int = 0) -> None:
    """pages[..., dst[i], ...] = pages[..., src[i], ...] for every i along dimension ``dim``, in place, one launch for each 448 pairs:
    ``pages`` is a cache's whole storage (any type), the page's own dimensions after ``dim`` contiguous, the dimensions
    before it (layers; keys and values) evenly spaced.  src and dst are page numbers on the host (lists,
    arrays or CPU tensors); a page outside of the cache, written twice, or both read and written raises ValueError and
    nothing is copied.  Under HIP graph capture the pairs of the capture are recorded."""
    what = "copy_pages"
    if _fast is not None and _unwatched() and _fast.copy_pages(pages, src, dst, dim):
        return
    ops._require_gpu(pages, what)
    dim = dim + pages.dim() if dim < 0 else dim
    if not 0 <= dim < pages.dim():
        raise ValueError(f"{what}: no dimension {dim} in {tuple(pages.shape)}")
    s, d = _pairs(src, what), _pairs(dst, what)
    if s.size != d.size:
        raise ValueError(f"{what}: {s.size} sources for {d.size} destinations")
    _, _, count, page, n = _layout(pages, dim)
    if _direct(pages):
        _copy_into(pages, s, d, dim)
        torch.autograd.graph.increment_version(pages)
    else:
        # of no plane: the pairs are looked at, and nothing is launched
        check(lib.gqk_copy_pages(None, 0, 0, count, page, n, s.ctypes.data, d.ctypes.data, s.size, None), what)
        _copy_op(pages, s.tolist(), d.tolist(), dim)


class PagePool:
    """Which of a cache's pages are in use, and by how many sequences.  Host bookkeeping alone: the methods that need
    pages copied return the (source, destination) pairs for ``copy_pages``.

        pool = PagePool(1024)
        table = pool.allocate(pages)                    # a sequence's pages
        child = pool.fork(table)                        # a second sequence on the same pages
        src, dst = pool.own(child, len(child) - 1)      # before it writes its last page: a page of its own
        copy_pages(storage, src, dst, dim=1)
        pool.free(table)
        src, dst = pool.compact([child])                # live pages to the front, tables renumbered
    """

    def __init__(self, pages: int):
        if pages < 0:
            raise ValueError(f"PagePool: {pages} pages")
        self.uses = [0] * pages          # sequences on each page
        self._free = list(range(pages))  # a heap: the lowest page first, so live pages stay together

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def allocate(self, n: int = 1) -> list[int]:
        """n pages of the caller's own, or MemoryError and none."""
        if n < 0:
            raise ValueError(f"PagePool: {n} pages")
        if n > len(self._free):
            raise MemoryError(f"PagePool: {n} pages wanted, {len(self._free)} of {len(self.uses)} free")
        got = [heapq.heappop(self._free) for _ in range(n)]
        for p in got:
            self.uses[p] = 1
        return got

    def _check(self, table) -> None:
        for p in table:
            if not 0 <= p < len(self.uses) or self.uses[p] == 0:
                raise ValueError(f"PagePool: page {p} is not in use")

    def fork(self, table) -> list[int]:
        """A second table on the same pages."""
        self._check(table)
        for p in table:
            self.uses[p] += 1
        return list(table)

    def own(self, table: list[int], i: int) -> tuple[list[int], list[int]]:
        """Makes table[i] a page that no other sequence reads, before it is written: the pairs to copy (none if it was)."""
        self._check([table[i]])
        old = table[i]
        if self.uses[old] == 1:
            return [], []
        new = self.allocate(1)[0]
        self.uses[old] -= 1
        table[i] = new
        return [old], [new]

    def free(self, table) -> None:
        """Gives up one use of each page; a page that nobody uses any more is free."""
        table = list(table)
        self._check(table)
        count: dict[int, int] = {}
        for p in table:
            count[p] = count.get(p, 0) + 1
        for p, c in count.items():
            if c > self.uses[p]:
                raise ValueError(f"PagePool: page {p} freed {c} times, used {self.uses[p]}")
        for p, c in count.items():
            self.uses[p] -= c
            if self.uses[p] == 0:
                heapq.heappush(self._free, p)

    def compact(self, tables: list[list[int]]) -> tuple[list[int], list[int]]:
        """Moves the live pages to the front of the cache: the pairs to copy.  ``tables`` are all tables on the pool,
        renumbered in place (a live page that none of them names is an error, and nothing changes)."""
        live = sum(1 for u in self.uses if u)
        named: dict[int, int] = {}
        for t in tables:
            for p in t:
                named[p] = named.get(p, 0) + 1
        if any(self.uses[p] != named.get(p, 0) for p in range(len(self.uses))) or any(
                not 0 <= p < len(self.uses) for p in named):
            raise ValueError("PagePool: compact needs every table on the pool")
        holes = [p for p in range(live) if not self.uses[p]]
        far = [p for p in range(live, len(self.uses)) if self.uses[p]]
        move = dict(zip(far, holes))
        for t in tables:
            t[:] = [move.get(p, p) for p in t]
        for s, d in move.items():
            self.uses[d], self.uses[s] = self.uses[s], 0
        self._free = list(range(live, len(self.uses)))
        return list(move), list(move.values())
