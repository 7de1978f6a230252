"""Pages of a cache on the move: copies between pages of a pool, pages gathered into one buffer
(snapshots, hand-off) and scattered from one (``csrc/pages.cu``; tables from ``host/page_plan.cpp``). A page id addresses the same
slot of every slab, and every call moves all of a page in one launch per 128 slabs."""
from __future__ import annotations

import ctypes

import torch

from .. import host_runtime
from . import _lib

_COPY, _GATHER, _SCATTER = 0, 1, 2


def _list(ids) -> list:
    return ids.tolist() if hasattr(ids, "tolist") else list(ids)


class PageSlabs:
    """The slabs of a pool, [pages, ...] each, apart in memory, in the order in which a buffer holds them. Page ids are host lists (or
    CPU tensors and arrays) and are checked: a page outside the pool, a destination of two sources or a source missing raises ``ValueError``
    and moves nothing. Slabs whose pages are empty are left out. The ids of small calls (106 copies, 320 pages) travel with the launch, which can
    be captured into a graph; longer tables are copied to the device first, which cannot."""

    def __init__(self, slabs: list[torch.Tensor]):
        if not slabs:
            raise ValueError("a pool without slabs has no pages")
        self.num_pages, self.device = int(slabs[0].shape[0]), slabs[0].device
        for t in slabs:
            if t.shape[0] != self.num_pages or t.device != self.device or not t.is_contiguous():
                raise ValueError("slabs have to be contiguous, on one device and of as many pages each")
        self.slabs = [t for t in slabs if t.numel()]
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in self.slabs)
        if any(end > start for (_, end), (start, _) in zip(spans, spans[1:])):
            raise ValueError("slabs have to lie apart: bytes that two of them share would move twice")
        self.page_bytes = [t[0].numel() * t.element_size() for t in self.slabs]
        self.bytes_per_page = sum(self.page_bytes)
        n = len(self.slabs)
        self._base = (ctypes.c_void_p * n)(*(t.data_ptr() for t in self.slabs))
        self._size = (ctypes.c_longlong * n)(*self.page_bytes)

    def _launch(self, job: int, table, n: int, chains: int = 0, buffer: torch.Tensor | None = None, first: int = 0, count: int | None = None) -> None:
        ints, far = int(table.size), None
        count = len(self.slabs) - first if count is None else count
        if n == 0 or count == 0:
            return
        if ints > _lib.load().mx_pages_inline_ints():          # longer tables go through device memory
            far = torch.from_numpy(table).to(self.device)
        _lib.launch_on(self.device, "mx_pages", job, ctypes.addressof(self._base) + 8 * first, ctypes.addressof(self._size) + 8 * first, count,
                       _lib.ptr(buffer), table.ctypes.data, _lib.ptr(far), ints, n, chains)

    def copy(self, src, dst) -> None:
        """Page ``dst[i]`` becomes what page ``src[i]`` was before the call, for all i; a page may be both."""
        table, n, chains = host_runtime.page_copies(_list(src), _list(dst), self.num_pages)
        if self.device.type != "cuda":
            pairs = torch.from_numpy(table[:2 * n]).long().view(n, 2)
            for t in self.slabs:
                t[pairs[:, 1]] = t[pairs[:, 0]]
            return
        self._launch(_COPY, table, n, chains)

    def gather(self, ids, out: torch.Tensor | None = None, first: int = 0, count: int | None = None) -> torch.Tensor:
        """The pages ``ids`` of ``count`` slabs from ``first`` on (all) as bytes: slab after slab, the pages of each in the given order."""
        table, sizes, total = self._buffer(ids, False, first, count)
        if out is None:
            out = torch.empty(total, dtype=torch.uint8, device=self.device)
        self._check_buffer(out, total)
        if self.device.type != "cuda":
            idx, at = torch.from_numpy(table).long(), 0
            for t, size in zip(self.slabs[first:], sizes):
                out[at:at + size * table.size].copy_(t[idx].reshape(-1).view(torch.uint8))
                at += size * table.size
        else:
            self._launch(_GATHER, table, int(table.size), buffer=out, first=first, count=len(sizes))
        return out

    def scatter(self, ids, data: torch.Tensor, first: int = 0, count: int | None = None) -> None:
        """Puts what :meth:`gather` returned for as many pages into the pages ``ids`` (each named once)."""
        table, sizes, total = self._buffer(ids, True, first, count)
        self._check_buffer(data, total)
        if self.device.type != "cuda":
            idx, at = torch.from_numpy(table).long(), 0
            for t, size in zip(self.slabs[first:], sizes):
                t[idx] = data[at:at + size * table.size].clone().view(t.dtype).view(table.size, *t.shape[1:])
                at += size * table.size
        else:
            self._launch(_SCATTER, table, int(table.size), buffer=data, first=first, count=len(sizes))

    def _buffer(self, ids, unique: bool, first: int, count: int | None):
        n = len(self.slabs)
        count = n - first if count is None else count
        if not (0 <= first <= n and 0 <= count <= n - first):
            raise ValueError(f"slabs {first} to {first + count} of {n}")
        table = host_runtime.page_ids(_list(ids), self.num_pages, unique)
        sizes = self.page_bytes[first:first + count]
        return table, sizes, sum(sizes) * int(table.size)

    def _check_buffer(self, t: torch.Tensor, total: int) -> None:
        if t.dtype != torch.uint8 or t.numel() != total or t.device != self.device or not t.is_contiguous():
            raise ValueError(f"the pages are {total} contiguous bytes on {self.device}")
