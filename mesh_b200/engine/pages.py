"""KV page allocator. Uses the native runtime (``mesh_b200._runtime``) when built, else a Python
free list with identical behaviour (lowest page ids first, double-free detection). A page may have several
holders (sessions forked from one another): ``share`` adds one, ``free`` takes one away."""
from __future__ import annotations

import heapq
from typing import List, Optional


class _PyPageAllocator:
    def __init__(self, num_pages: int, reserved: int = 0):
        if num_pages <= reserved:
            raise ValueError("page pool too small")
        self.num_pages = num_pages
        self.reserved = reserved
        self._free = list(range(reserved, num_pages))
        heapq.heapify(self._free)
        self._used = {}  # page -> holders

    def alloc(self, n: int) -> Optional[List[int]]:
        if n > len(self._free):
            return None
        out = [heapq.heappop(self._free) for _ in range(n)]
        self._used.update((p, 1) for p in out)
        return out

    def free(self, pages: List[int]) -> None:
        for p in pages:
            if p not in self._used:
                raise ValueError(f"double free or foreign page {p}")
            self._used[p] -= 1
            if self._used[p] == 0:
                del self._used[p]
                heapq.heappush(self._free, p)

    def share(self, pages: List[int]) -> None:
        """One more holder for each of these pages; every holder frees them once."""
        for p in pages:
            if p not in self._used:
                raise ValueError(f"page {p} is not in use")
        for p in pages:
            self._used[p] += 1

    def refs(self, page: int) -> int:
        return self._used.get(page, 0)

    def remap(self, remap: List[int]) -> None:
        """After a compaction of the pool: page p is now remap[p]. Holders keep their counts; other pages are free."""
        if len(remap) != self.num_pages:
            raise ValueError("remap must cover the pool")
        moved = {}
        for p, n in self._used.items():
            q = remap[p]
            if not self.reserved <= q < self.num_pages:
                raise ValueError(f"page {p} is in use but has no new place")
            if q in moved:
                raise ValueError(f"two pages moved to {q}")
            moved[q] = n
        self._used = moved
        self._free = [p for p in range(self.reserved, self.num_pages) if p not in moved]

    @property
    def num_free(self) -> int:
        return len(self._free)

    @property
    def num_used(self) -> int:
        return len(self._used)


def PageAllocator(num_pages: int, reserved: int = 0):
    try:
        from .. import _runtime  # type: ignore
        return _runtime.PageAllocator(num_pages, reserved)
    except ImportError:
        return _PyPageAllocator(num_pages, reserved)
