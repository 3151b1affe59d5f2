"""Pages of a cache of states: copy, fork, reorder, compact and clear them, in place.

A page is row ``i`` along the first dimension of every tensor of a list: the Canon states of all layers and positions,
their write positions, linear attention states; that is, all that belongs to one request or beam.  One launch moves
the pages of up to 128 tensors, whatever their dtypes and page sizes.  Pages are moved as if all were read before any
is written: page ``i`` afterwards holds what its source held before the call, however the moves chain or cross.

``PageTable(states)`` checks the tensors once and offers the operations as methods; the functions build one per call.
Index tensors live on the device of the states.  An index outside ``0..pages-1`` moves nothing.
"""
from __future__ import annotations

import ctypes as C
from array import array
from itertools import repeat
from operator import attrgetter
from typing import Iterable, Tuple

import torch

from . import _cabi
from .ops import _no_tangents, _stream_handle

_nbytes, _requires_grad = attrgetter("nbytes"), attrgetter("requires_grad")
_INDEX_DTYPES = {torch.int32: _cabi.VC1D_I32, torch.int64: _cabi.VC1D_I64}


def _check_apart(table, pages: int) -> None:
    """Refuses tensors ``(address, bytes of a page, bytes from page to page)`` that share a byte."""
    ends = sorted((base, base + (pages - 1) * stride + size, size, stride) for base, size, stride in table if size > 0 and pages > 0)
    open_ = []  # tensors that reach beyond the start of the next one: the layers of one pool
    for a in ends:
        open_ = [b for b in open_ if b[1] > a[0]]
        for b in open_:
            d = (a[0] - b[0]) % a[3]
            if a[3] != b[3] or d < b[2] or d + a[2] > a[3]:  # equal strides: the pages interleave, or not
                raise ValueError("states overlap: a tensor is given twice, or two share memory")
        open_.append(a)


class PageTable:
    """The pages of ``states``: tensors on one CUDA device with the same first dimension, each page contiguous (the
    distance between pages is free, so the layers of a pool ``[pages, layers, ...]`` may be given one by one), none
    overlapping another.  The table names their memory: build a new one after a state was replaced."""

    def __init__(self, states: Iterable[torch.Tensor]):
        self.states = list(states)
        _no_tangents("moving pages", *self.states)
        self.device = self.states[0].device if self.states else None
        self.pages = int(self.states[0].shape[0]) if self.states and self.states[0].dim() else 0
        # three numbers a tensor: address, bytes of a page, bytes from page to page.  A model's cache has many small
        # states, so the common case asks each attribute of all of them at once.
        table = array("q", bytes(24 * len(self.states)))
        index = self.device.index if self.states else None
        if (self.pages > 0 and self.device.type == "cuda" and all(map(torch.Tensor.is_contiguous, self.states)) and all(map(index.__eq__, map(torch.Tensor.get_device, self.states)))
                and all(map(torch.Tensor.dim, self.states)) and all(map(self.pages.__eq__, map(torch.Tensor.size, self.states, repeat(0))))
                and not (torch.is_grad_enabled() and any(map(_requires_grad, self.states)))):
            table[0::3] = array("q", map(torch.Tensor.data_ptr, self.states))
            table[1::3] = table[2::3] = array("q", map(self.pages.__rfloordiv__, map(_nbytes, self.states)))
        else:
            for n, t in enumerate(self.states):
                table[3 * n: 3 * n + 3] = array("q", self._strided(t))
        self._table = table
        if len(self.states) > _cabi.PAGES_MAX_TENSORS:  # a launch looks at its own tensors only
            _check_apart(list(zip(table[0::3], table[1::3], table[2::3])), self.pages)
        if self.pages > _cabi.PAGES_MAX_PAGES:
            raise ValueError(f"at most {_cabi.PAGES_MAX_PAGES} pages, got {self.pages}")

    def _strided(self, t: torch.Tensor):
        if t.dim() < 1:
            raise ValueError("a state needs a first dimension: its pages")
        if t.device.type != "cuda":
            raise ValueError(f"a state must be on a CUDA device, got {t.device}")
        if t.device != self.device:
            raise ValueError(f"a state is on {t.device}, the first on {self.device}")
        if t.shape[0] != self.pages:
            raise ValueError(f"a state has {t.shape[0]} pages, the first {self.pages}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError("a state requires grad: pages are moved in place")
        item, inner = t.element_size(), 1
        for size, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
            if size > 1 and stride != inner:
                raise ValueError(f"a page must be contiguous, got strides {t.stride()}")
            inner *= size
        if self.pages > 1 and t.stride(0) < inner:
            raise ValueError(f"pages overlap: stride {t.stride(0)} for {inner} values")
        return t.data_ptr(), inner * item, (t.stride(0) if self.pages > 1 else inner) * item

    def _run(self, op: int, source=None, dst=None, n: int = 0, live=None, new_index=None, count=None) -> None:
        a = _cabi.PagesArgs()
        a.struct_size = C.sizeof(_cabi.PagesArgs)
        a.op, a.pages, a.n = op, self.pages, n
        for name, t in (("source", source), ("dst", dst), ("live", live), ("new_index", new_index), ("count", count)):
            if t is not None:
                setattr(a, name, t.data_ptr())
        index = source if source is not None else dst
        if len(self.states) > _cabi.PAGES_MAX_TENSORS:  # refused before the first launch, not between two
            self._check_arrays([t for t in (source, dst, live) if t is not None])
        if index is not None:
            a.index_dtype = _INDEX_DTYPES[index.dtype]
        stream = _stream_handle(self.device)
        base, size, total = self._table.buffer_info()[0], C.sizeof(_cabi.PageTensor), len(self.states)
        other = self.device.index != torch.cuda.current_device()
        if other:
            prev = torch.cuda.current_device()
            torch.cuda.set_device(self.device)
        try:
            for first in range(0, total, _cabi.PAGES_MAX_TENSORS):
                a.n_tensors = min(_cabi.PAGES_MAX_TENSORS, total - first)
                a.tensors = C.cast(base + first * size, C.POINTER(_cabi.PageTensor))
                st = _cabi.lib.vc1d_pages(C.byref(a), stream)
                if st != 0:
                    _cabi.check(st, "cache pages")
        finally:
            if other:
                torch.cuda.set_device(prev)
        torch.autograd.graph.increment_version(self.states)  # a graph that saved one of them refuses to run

    def _check_arrays(self, arrays) -> None:
        table = self._table
        for t in arrays:
            lo, hi = t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()
            for base, size, stride in zip(table[0::3], table[1::3], table[2::3]):
                if size > 0 and lo < base + (self.pages - 1) * stride + size and base < hi:
                    raise ValueError("an index tensor lies among the pages that are moved")

    def _index(self, t: torch.Tensor, what: str) -> torch.Tensor:
        if not isinstance(t, torch.Tensor) or t.dim() != 1:
            raise ValueError(f"{what} must be a 1D tensor")
        if t.dtype not in _INDEX_DTYPES:
            raise ValueError(f"{what} must be int32 or int64, got {t.dtype}")
        if t.shape[0] > _cabi.PAGES_MAX_ENTRIES:
            raise ValueError(f"{what} has {t.shape[0]} entries, at most {_cabi.PAGES_MAX_ENTRIES}")
        if self.device is not None and t.device != self.device:
            raise ValueError(f"{what} is on {t.device}, the states on {self.device}")
        return t.contiguous()

    def reorder(self, source: torch.Tensor) -> None:
        """Page ``i`` takes over page ``source[i]`` (beam search; a page may be taken by several); ``source[i] == i``
        costs nothing."""
        source = self._index(source, "source")
        if source.shape[0] != self.pages and self.states:
            raise ValueError(f"source has {source.shape[0]} entries for {self.pages} pages")
        if self.states:
            self._run(_cabi.PAGES_REORDER, source=source)

    def copy(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Page ``dst[i]`` takes over page ``src[i]``; a fork names one source several times.  Of equal destinations
        the first entry counts."""
        src, dst = self._index(src, "src"), self._index(dst, "dst")
        if src.shape != dst.shape or src.dtype != dst.dtype:
            raise ValueError("src and dst must have the same length and dtype")
        if self.states and src.numel():
            self._run(_cabi.PAGES_COPY, source=src, dst=dst, n=src.numel())

    def free(self, pages: torch.Tensor) -> None:
        """Clears the given pages to zero, as a new request finds them."""
        pages = self._index(pages, "pages")
        if self.states and pages.numel():
            self._run(_cabi.PAGES_FREE, dst=pages, n=pages.numel())

    def compact(self, live: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """Moves the live pages (``live[pages]``, bool or uint8) to the front: with n of them, the free pages below n
        take, in order, the live pages from n on.  Live pages below n stay where they are, what lies from n on is left
        as it is.  Returns ``new_index[pages]`` (int32: where each page is afterwards, -1 if it was free) and
        ``count[1]`` (int32: n), both on the device; nothing waits for the GPU."""
        if not self.states:
            raise ValueError("no states to compact")
        if live.dtype not in (torch.bool, torch.uint8) or tuple(live.shape) != (self.pages,):
            raise ValueError(f"live must be bool or uint8 [{self.pages}], got {live.dtype} {tuple(live.shape)}")
        if live.device != self.device:
            raise ValueError(f"live is on {live.device}, the states on {self.device}")
        live = live.contiguous()
        maps = torch.empty(self.pages + 1, dtype=torch.int32, device=self.device)
        new_index, count = maps[: self.pages], maps[self.pages:]
        self._run(_cabi.PAGES_COMPACT, live=live, new_index=new_index, count=count)
        return new_index, count


def reorder_pages(states: Iterable[torch.Tensor], source: torch.Tensor) -> None:
    """``PageTable(states).reorder(source)``: beam search over a cache, in place and in one launch."""
    PageTable(states).reorder(source)


def copy_pages(states: Iterable[torch.Tensor], src: torch.Tensor, dst: torch.Tensor) -> None:
    """``PageTable(states).copy(src, dst)``: copies pages, or forks one into several."""
    PageTable(states).copy(src, dst)


def free_pages(states: Iterable[torch.Tensor], pages: torch.Tensor) -> None:
    """``PageTable(states).free(pages)``: clears pages to zero."""
    PageTable(states).free(pages)


def compact_pages(states: Iterable[torch.Tensor], live: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``PageTable(states).compact(live)``: moves the live pages to the front; returns ``(new_index, count)``."""
    return PageTable(states).compact(live)
