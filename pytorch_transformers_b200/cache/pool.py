"""Host-side bookkeeping of the cache: which pages and which sequence slots are in use.

Pure Python, no device memory: the invariants (no page lost, held twice or freed twice; no
slot given out twice) are checked here and tested without a GPU.
"""
from __future__ import annotations

import heapq
from typing import Dict, List


class CacheFull(RuntimeError):
    """More tokens were asked for than the cache was sized for."""


class CacheError(RuntimeError):
    """Misuse of the cache: a page or slot freed twice, an unknown slot, and the like."""


class IdPool:
    """Integer ids 0 .. capacity-1, handed out lowest first and taken back. An id that is out may be shared: it goes back to the
    free ones when every holder has given it back."""

    def __init__(self, capacity: int, what: str):
        if capacity < 0:
            raise ValueError(f"{what} capacity must be >= 0, got {capacity}")
        self.capacity = capacity
        self.what = what
        self._free: List[int] = list(range(capacity))
        heapq.heapify(self._free)
        self._held = [0] * capacity     # holders of each id

    @property
    def available(self) -> int:
        return len(self._free)

    @property
    def in_use(self) -> int:
        return self.capacity - len(self._free)

    def take(self, n: int = 1) -> List[int]:
        if n < 0:
            raise ValueError("cannot take a negative number of ids")
        if n > len(self._free):
            raise CacheFull(f"{n} more {self.what}(s) needed but only {len(self._free)} of {self.capacity} are free")
        out = [heapq.heappop(self._free) for _ in range(n)]
        for i in out:
            if self._held[i]:
                raise CacheError(f"{self.what} {i} was in the free list while held")  # never expected
            self._held[i] = 1
        return out

    def _must_be_out(self, ids) -> None:
        for i in ids:
            if not (0 <= i < self.capacity):
                raise CacheError(f"{self.what} {i} is outside 0..{self.capacity - 1}")
            if not self._held[i]:
                raise CacheError(f"{self.what} {i} is freed twice (or was never given out)")

    def share(self, ids) -> None:
        """One more holder for each of ``ids``, which are out."""
        ids = list(ids)
        self._must_be_out(ids)
        for i in ids:
            self._held[i] += 1

    def holders(self, i: int) -> int:
        return self._held[i]

    def give_back(self, ids) -> None:
        ids = list(ids)
        self._must_be_out(ids)
        if len(set(ids)) != len(ids):
            raise CacheError(f"a {self.what} is named twice in one release: {ids}")
        for i in ids:
            self._held[i] -= 1
            if self._held[i] == 0:
                heapq.heappush(self._free, i)

    def renumber(self, capacity: int) -> Dict[int, int]:
        """Give the ids that are out new numbers 0 .. in_use-1 in a pool of ``capacity``: those below in_use keep theirs, the others
        take the lowest free ones. Returns {old: new} of the ids that changed."""
        n = self.in_use
        if capacity < n:
            raise CacheFull(f"{n} {self.what}s are out, more than a capacity of {capacity}")
        holes = [i for i in range(n) if not self._held[i]]
        moved = dict(zip((i for i in range(n, self.capacity) if self._held[i]), holes))
        held = self._held[:n]
        for old, new in moved.items():
            held[new] = self._held[old]
        self.capacity = capacity
        self._held = held + [0] * (capacity - n)
        self._free = list(range(n, capacity))      # sorted: a heap
        return moved

    def grow(self, capacity: int) -> None:
        """More ids, behind those that there are."""
        for i in range(self.capacity, capacity):
            self._held.append(0)
            heapq.heappush(self._free, i)
        self.capacity = max(self.capacity, capacity)

    def check(self) -> None:
        """Every id is either free or held, exactly once."""
        free = sorted(self._free)
        if len(set(free)) != len(free):
            raise CacheError(f"a {self.what} is twice in the free list")
        held = [i for i, h in enumerate(self._held) if h]
        if sorted(free + held) != list(range(self.capacity)):
            raise CacheError(f"{self.what} ids are lost or duplicated: free={free} held={held}")


class SequenceRecord:
    """What one live sequence holds: its length and, for each storage group, its pages.
    ``pages[g][i]`` holds positions [page_size*i, page_size*(i+1)); -1 marks a page that a
    window group has already released."""
    __slots__ = ("length", "pages")

    def __init__(self, n_groups: int):
        self.length = 0
        self.pages: List[List[int]] = [[] for _ in range(n_groups)]
