"""Host-side bookkeeping of what the cache hands out: sequence slots and pages.

Nothing here touches a device.  A handle that is given back twice, or that was
never handed out, is an error, so a leak or a double free shows at once.
"""
from __future__ import annotations

from collections import Counter
from typing import List


class CacheFull(RuntimeError):
    """The cache has no free slot or not enough free pages for the request."""


class HandleError(RuntimeError):
    """A slot or page was freed twice, or was never handed out."""


class FreeList:
    """Integers 0..n-1; lowest free number first, so runs are reproducible.  A number may be held several times over (``share``);
    it is free again when it has been given back as often."""

    def __init__(self, n: int, what: str):
        self.n = int(n)
        self.what = what
        self._free: List[int] = list(range(self.n - 1, -1, -1))   # pop() gives the lowest
        self._held = [0] * self.n              # how many times over

    @property
    def n_free(self) -> int:
        return len(self._free)

    @property
    def n_held(self) -> int:
        return self.n - len(self._free)

    def take(self, count: int = 1) -> List[int]:
        if count > len(self._free):
            raise CacheFull(f"{count} {self.what}(s) wanted, {len(self._free)} of {self.n} free")
        out = [self._free.pop() for _ in range(count)]
        for i in out:
            self._held[i] = 1
        return out

    def share(self, handles) -> None:
        """Holds the handles, which are held already, once more."""
        handles = list(handles)
        for i in handles:
            if not self.is_held(i):
                raise HandleError(f"{self.what} {i} is not held and cannot be shared")
        for i in handles:
            self._held[i] += 1

    def move(self, moves) -> None:
        """Every (held, free) pair changes places."""
        for a, b in moves:
            if not self.is_held(a) or not 0 <= b < self.n or self._held[b]:
                raise HandleError(f"{self.what} {a} cannot move to {b}")
            self._held[b], self._held[a] = self._held[a], 0
        self._free = [i for i in range(self.n - 1, -1, -1) if not self._held[i]]

    def times_held(self, i: int) -> int:
        return self._held[i]

    def give_back(self, handles) -> None:
        handles = list(handles)
        times = Counter(handles)
        for i, n in times.items():
            if not (0 <= i < self.n) or self._held[i] < n:
                raise HandleError(f"{self.what} {i} is not held (freed twice, or never handed out)")
        for i, n in times.items():
            self._held[i] -= n
        self._free.extend(i for i in times if not self._held[i])
        self._free.sort(reverse=True)

    def is_held(self, i: int) -> bool:
        return 0 <= i < self.n and self._held[i] > 0
