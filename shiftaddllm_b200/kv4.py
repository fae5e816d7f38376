"""Pages of a 4-bit cache: which sequence has which, on the host.

The pool (:func:`decode_ops.kv4_pool`) holds pages of 64 positions of all layers; a sequence (`slot`) has a list of them, in the device table
that the kernels read.  Pages are counted: a forked sequence shares its parent's, and whoever first writes into a shared page gets a copy of its
own.  All calls act in the order of torch's current stream, so pages that earlier launches read may be given away at once; with several
streams the caller orders them.
"""
from __future__ import annotations

import heapq

import torch

from . import decode_ops

PAGE = decode_ops.KV4_PAGE


class Kv4Cache:
    """Keys and values of up to `slots` sequences of up to `max_len` positions, in `pages` pages shared by all.

    ``pool[layer]`` and ``table`` are what :func:`decode_ops.rope_kv4_write`, :func:`decode_ops.attention_kv4` and :func:`decode_ops.read_kv4`
    take; both stay where they are for as long as the cache lives, so captured launches go on seeing it."""

    def __init__(self, layers: int, kv_heads: int, hd: int, slots: int, max_len: int, pages: int | None = None, device="cuda"):
        if min(layers, kv_heads, slots, max_len) < 1 or (pages is not None and pages < 1):
            raise ValueError("layers, kv_heads, slots, max_len and pages must be at least 1")
        self.kv_heads, self.hd, self.max_len = kv_heads, hd, max_len
        width = -(-max_len // PAGE)
        self.pages = slots * width if pages is None else pages
        self.pool = decode_ops.kv4_pool(layers, self.pages, kv_heads, hd, device)
        self.table = torch.full((slots, width), -1, dtype=torch.int32, device=device)      # -1: a page that does not exist
        self._of = [[] for _ in range(slots)]            # pages of each slot, in order
        self._users = [0] * self.pages
        self._free = list(range(self.pages))             # a heap: the lowest page first

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def pages_of(self, slot: int) -> list[int]:
        return list(self._pages(slot))

    def _pages(self, slot: int) -> list[int]:
        if not 0 <= slot < len(self._of):      # a list would count negative ones from its end: two names for one sequence
            raise ValueError(f"there is no sequence {slot} of {len(self._of)}")
        return self._of[slot]

    def _take(self, n: int) -> list[int]:
        if n > len(self._free):
            raise RuntimeError(f"the cache has {len(self._free)} free pages, {n} are needed")
        got = [heapq.heappop(self._free) for _ in range(n)]
        for p in got:
            self._users[p] = 1
        return got

    def _drop(self, page: int) -> None:
        self._users[page] -= 1
        if self._users[page] == 0:
            heapq.heappush(self._free, page)

    def _publish(self, *slots: int) -> None:
        width = self.table.shape[1]
        for s in slots:
            self.table[s].copy_(torch.tensor(self._of[s] + [-1] * (width - len(self._of[s])), dtype=torch.int32))

    def reserve(self, slot: int, first: int, last: int) -> None:
        """Makes positions first .. last - 1 of a sequence writable: pages it lacks are added, pages it shares with others in that range are
        replaced by copies.  RuntimeError, and nothing changed, where there are not enough free pages."""
        self.reserve_all([(slot, first, last)])

    def reserve_all(self, ranges) -> None:
        """:meth:`reserve` for several sequences, `ranges` of (slot, first, last): all of them, or none."""
        plan, users, need, slots = [], {}, 0, set()
        for slot, first, last in ranges:
            if not 0 <= first <= last <= self.max_len:
                raise ValueError(f"positions {first} .. {last} of {self.max_len}")
            mine = self._pages(slot)
            if first > len(mine) * PAGE:
                raise ValueError(f"position {first} lies behind the sequence's {len(mine)} pages")
            if slot in slots:
                raise ValueError(f"sequence {slot} stands in the list twice")
            slots.add(slot)
            width = -(-last // PAGE)
            shared = []
            for i in range(first // PAGE, min(width, len(mine))) if last > first else ():
                left = users.get(mine[i], self._users[mine[i]])      # the last of its users keeps the page
                if left > 1:
                    shared.append(i)
                    users[mine[i]] = left - 1
            more = max(0, width - len(mine))
            plan.append((slot, shared, more))
            need += len(shared) + more
        if need == 0:
            return
        got = self._take(need)
        into, src, dst = iter(got), [], []
        new = {}
        for slot, shared, more in plan:
            pages = new[slot] = list(self._of[slot])
            for i in shared:
                src.append(pages[i])
                pages[i] = next(into)
                dst.append(pages[i])
            pages += [next(into) for _ in range(more)]
        try:
            decode_ops.copy_kv4_pages(self.pool, src, dst)
        except BaseException:
            for p in got:
                self._drop(p)
            raise
        for p in src:
            self._drop(p)
        changed = [slot for slot, shared, more in plan if shared or more]
        for slot in changed:
            self._of[slot] = new[slot]
        self._publish(*changed)

    def fork(self, src: int, dst: int) -> None:
        """Sequence `dst` (whose own pages are given up) becomes one with `src`'s positions; the pages are shared until one of them writes."""
        pages = list(self._pages(src))
        self._pages(dst)
        if src == dst:
            return
        for p in pages:
            self._users[p] += 1
        self._give_up(dst, 0)
        self._of[dst] = pages
        self._publish(dst)

    def truncate(self, slot: int, length: int) -> None:
        """Gives up the pages behind position length - 1."""
        if length < 0:
            raise ValueError("length must not be negative")
        self._pages(slot)
        self._give_up(slot, -(-length // PAGE))
        self._publish(slot)

    def free(self, slot: int) -> None:
        self.truncate(slot, 0)

    def _give_up(self, slot: int, keep: int) -> None:
        for p in self._of[slot][keep:]:
            self._drop(p)
        del self._of[slot][keep:]

    def compact(self) -> int:
        """Moves the used pages to the front of the pool; returns their number.  What lies behind them is free."""
        used = self.pages - len(self._free)
        moves = {}
        holes = sorted(p for p in self._free if p < used)
        for p in range(used, self.pages):
            if self._users[p]:
                moves[p] = holes[len(moves)]
        if moves:
            decode_ops.copy_kv4_pages(self.pool, list(moves), list(moves.values()))
            for a, b in moves.items():
                self._users[b], self._users[a] = self._users[a], 0
            touched = []
            for s, mine in enumerate(self._of):
                if any(p in moves for p in mine):
                    self._of[s] = [moves.get(p, p) for p in mine]
                    touched.append(s)
            self._free = list(range(used, self.pages))
            heapq.heapify(self._free)
            self._publish(*touched)
        return used
