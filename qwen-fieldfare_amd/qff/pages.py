"""Bookkeeping of a paged KV cache on the host: which page of the pools holds
which positions of which sequence.

One PageTable serves all full-attention layers of a model: page i is page i of
every layer's K and V pool. Sequences live in slots, the rows of the device
tables that gqa_decode_paged / gqa_decode_shared / gqa_prefill_paged read.
Pages are counted: forked sequences hold their parent's pages until one of the
holders writes into one, which then gets a page of its own (copy on write).

The table changes here; the pages themselves are copied by the caller, with
ops.pages_copy over its pools and the pairs that reserve() and compact() return,
before the next call that reads or writes them. The device tensors `table`,
`group` and `shared_len` are updated in place by sync(), so a captured decode
step goes on using them.

No counterpart in the reference, which keeps one flat cache per layer for its
one sequence (QwenQ4ActiveExpertStreamingRunner.swift:726-742).
"""
from __future__ import annotations

import heapq

import numpy as np
import torch


class OutOfPages(RuntimeError):
    """The pool has fewer free pages than a call needs; nothing was changed."""


class PageTable:
    # shorter shared prefixes are not grouped (the attention reads them per sequence too)
    MIN_SHARED = 64

    def __init__(self, num_pages: int, page_size: int, slots: int, max_ctx: int, device="cuda"):
        if num_pages <= 0 or slots <= 0 or max_ctx <= 0:
            raise ValueError("num_pages, slots and max_ctx must be positive")
        if page_size < 16 or page_size > 4096 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two, 16 .. 4096")
        self.page_size = page_size
        self.cols = -(-max_ctx // page_size)
        self.lengths = [0] * slots                      # positions each slot holds
        self.refs = np.zeros(num_pages, np.int64)       # holders of each page
        self._free = list(range(num_pages))             # a heap: the lowest page first
        self._rows = np.full((slots, self.cols), -1, np.int32)
        dev = dict(dtype=torch.int32, device=device)
        self.table = torch.full((slots, self.cols), -1, **dev)
        self.group = torch.full((slots,), -1, **dev)
        self.shared_len = torch.zeros(slots, **dev)
        self._dirty = False

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def check_slot(self, slot: int) -> None:
        """Refuses what is no slot's number (a negative one would be another slot's)."""
        if not 0 <= slot < len(self.lengths):
            raise IndexError(f"slot {slot} of {len(self.lengths)}")

    def pages_of(self, slot: int) -> list[int]:
        self.check_slot(slot)
        return [int(p) for p in self._rows[slot, :-(-self.lengths[slot] // self.page_size)]]

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self.refs[page] = 1
        return page

    def _drop(self, page: int):
        self.refs[page] -= 1
        if self.refs[page] == 0:
            heapq.heappush(self._free, int(page))

    def reserve(self, slot: int, start: int, end: int) -> list[tuple[int, int]]:
        """Positions start .. end - 1 of `slot` are about to be written: gives
        it pages of its own for them. Returns the (source, destination) pages to
        copy in every pool first, for pages it shared and that hold positions it
        keeps. Positions before start must be there already."""
        self.check_slot(slot)
        if not 0 <= start < end or start > self.lengths[slot]:
            raise ValueError(f"positions {start} .. {end - 1} do not follow the {self.lengths[slot]} that slot {slot} holds")
        if end > self.cols * self.page_size:
            raise ValueError(f"slot {slot}: {end} positions do not fit {self.cols} pages")
        row, first, last = self._rows[slot], start // self.page_size, (end - 1) // self.page_size
        new = [c for c in range(first, last + 1) if row[c] < 0 or self.refs[row[c]] > 1]
        if len(new) > len(self._free):
            raise OutOfPages(f"{len(new)} pages needed, {len(self._free)} free")
        copies = []
        for c in new:
            old, page = int(row[c]), self._take()
            if old >= 0:
                # positions of the page that are kept: before start, or past end
                if c * self.page_size < start or min((c + 1) * self.page_size, self.lengths[slot]) > end:
                    copies.append((old, page))
                self._drop(old)
            row[c] = page
            self._dirty = True
        self.lengths[slot] = max(self.lengths[slot], end)
        return copies

    def fork(self, src: int, dst: int) -> None:
        """Slot dst (empty) gets what slot src holds; no page is copied."""
        self.check_slot(src)
        self.check_slot(dst)
        if src == dst or self.lengths[dst]:
            raise ValueError(f"slot {dst} must be empty")
        n = -(-self.lengths[src] // self.page_size)
        self._rows[dst, :n] = self._rows[src, :n]
        for page in self._rows[src, :n]:
            self.refs[page] += 1
        self.lengths[dst] = self.lengths[src]
        self._dirty = True

    def release(self, slot: int) -> None:
        """Empties a slot; pages that no other slot holds are free again."""
        for page in self.pages_of(slot):
            self._drop(page)
        self._rows[slot] = -1
        self.lengths[slot] = 0
        self._dirty = True

    def truncate(self, slot: int, end: int) -> None:
        """Slot `slot` holds its first `end` positions only: a reservation taken
        back, or tokens that are given up (recurrent states are the caller's). Pages
        behind them that no other slot holds are free again."""
        self.check_slot(slot)
        if not 0 <= end <= self.lengths[slot]:
            raise ValueError(f"slot {slot} holds {self.lengths[slot]} positions, not {end}")
        if end == self.lengths[slot]:
            return
        row, keep = self._rows[slot], -(-end // self.page_size)
        for page in self.pages_of(slot)[keep:]:
            self._drop(page)
        row[keep:] = -1
        self.lengths[slot] = end
        self._dirty = True

    def compact(self) -> tuple[list[int], list[int]]:
        """Moves the pages in use to the front of the pools: returns sources
        and destinations (disjoint) of the copies to make in every pool. Pages
        from the number in use on are then free."""
        live = np.flatnonzero(self.refs)
        n = len(live)
        src = live[live >= n]
        dst = np.flatnonzero(self.refs[:n] == 0)
        if len(src):
            moved = np.arange(len(self.refs), dtype=np.int32)
            moved[src] = dst
            held = self._rows >= 0
            self._rows[held] = moved[self._rows[held]]
            self.refs[dst] = self.refs[src]
            self.refs[src] = 0
            self._free = list(range(n, len(self.refs)))
            self._dirty = True
        return [int(p) for p in src], [int(p) for p in dst]

    def groups(self) -> tuple[np.ndarray, np.ndarray]:
        """(group, shared_len) of every slot, from the pages that neighbouring
        slots share from the start: a slot joins the group of the slots before it
        where it shares at least MIN_SHARED positions with the first of them and
        at least half of what they share."""
        n = len(self.lengths)
        group, shared = np.full(n, -1, np.int32), np.zeros(n, np.int32)
        first = 0
        for b in range(1, n + 1):
            common = 0
            if b < n and self.lengths[b] and self.lengths[first]:
                same = (self._rows[b] == self._rows[first]) & (self._rows[b] >= 0)
                common = (self.cols if same.all() else int(same.argmin())) * self.page_size
                common = min(common, self.lengths[b], self.lengths[first])
            if b > first + 1:
                least = int(shared[first + 1:b].min())
            else:
                least = 0
            if common >= self.MIN_SHARED and 2 * common >= least:
                shared[b] = common
                continue
            if b > first + 1:   # slots first .. b - 1 are a group
                shared[first] = least
                group[first:b] = first
            first = b
        return group, shared

    def sync(self) -> None:
        """Brings the device tensors up to date, where anything changed."""
        if not self._dirty:
            return
        group, shared = self.groups()
        self.table.copy_(torch.from_numpy(self._rows))
        self.group.copy_(torch.from_numpy(group))
        self.shared_len.copy_(torch.from_numpy(shared))
        self._dirty = False
