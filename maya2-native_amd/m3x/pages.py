"""Pages of a paged KV cache: which page holds which positions of which slot (host side), and the device table that
says so to the kernels (ops.PagedKv, one table for all layers).

A slot's positions live in pages of page_size positions, taken from a pool as the slot grows. Slots may share pages (a
prefix installed once): a page is free again when the last slot that names it lets go. Pages are only ever written by
the one slot that took them new, so shared ones never change. Changes to the table are collected on the host and sent
by `flush`, in stream order before the step that needs them."""
from __future__ import annotations

from contextlib import contextmanager

import numpy as np
import torch

from .staging import Upload


class PagePool:
    SEND = 4096  # table entries a copy

    def __init__(self, pages, page_size, slots, capacity, device):
        if pages < 1 or slots < 1 or capacity < 1:
            raise ValueError(f"PagePool: {pages} pages for {slots} slots of {capacity} positions")
        self.pages, self.page_size, self.slots = int(pages), int(page_size), int(slots)
        self.width = -(-int(capacity) // self.page_size)
        self.table = torch.full((self.slots, self.width), -1, dtype=torch.int32, device=device)
        self._host = np.full((self.slots, self.width), -1, dtype=np.int32)
        self._uses = np.zeros(self.pages, dtype=np.int32)  # slots that name a page
        self._free = list(range(self.pages - 1, -1, -1))
        self._end = [0] * self.slots    # table entries a slot has taken so far (some may be released again)
        self._begin = [0] * self.slots  # first entry behind those that were released
        self._changed = {}              # flat table index -> page, not yet sent
        self._index = self._value = None
        self._log = None                # within an attempt: (slot, entry, page before) of each change

    @property
    def free_pages(self):
        return len(self._free)

    def _check(self, *slots):
        for slot in slots:
            if not 0 <= slot < self.slots:
                raise IndexError(f"slot {slot} outside 0..{self.slots - 1}")

    def held(self, slot):
        """Pages that the slot names."""
        self._check(slot)
        return int((self._host[slot] >= 0).sum())

    def has(self, slot, length):
        """Whether the slot's first `length` positions all lie in pages."""
        self._check(slot)
        end = -(-int(length) // self.page_size)
        return end <= self.width and bool((self._host[slot, :max(end, 0)] >= 0).all())

    @contextmanager
    def attempt(self, keep=True):
        """Changes that belong together (none of them sent in between): where one of them raises, all are taken back; without
        keep in any case, to see whether one does."""
        kept = list(self._end), list(self._begin), dict(self._changed)
        log = self._log = []
        try:
            yield
        except BaseException:
            keep = False
            raise
        finally:
            self._log = None
            if not keep:
                self._undo(log, *kept)

    def _undo(self, log, end, begin, changed):
        """The log's changes backwards: pages go back to the free ones' top, and come from there, in the opposite order."""
        for slot, at, page in reversed(log):
            taken = int(self._host[slot, at])
            if taken >= 0:
                self._uses[taken] -= 1
                if self._uses[taken] == 0:
                    self._free.append(taken)
            if page >= 0:
                if self._uses[page] == 0:
                    self._free.pop()
                self._uses[page] += 1
            self._host[slot, at] = page
        self._end, self._begin, self._changed = end, begin, changed

    def _set(self, slot, at, page):
        if self._log is not None:
            self._log.append((slot, at, int(self._host[slot, at])))
        self._host[slot, at] = page
        self._changed[slot * self.width + at] = page

    def _drop(self, slot, at):
        page = int(self._host[slot, at])
        if page >= 0:
            self._uses[page] -= 1
            if self._uses[page] == 0:
                self._free.append(page)
            self._set(slot, at, -1)

    def grow(self, wants):
        """wants: (slot, length) pairs. Takes the pages that the slots' first `length` positions still need; RuntimeError,
        with nothing taken, when the pool has too few."""
        todo, ends = [], {}
        for slot, length in wants:
            self._check(slot)
            end = -(-int(length) // self.page_size)
            if end > self.width:
                raise ValueError(f"slot {slot}: {length} positions exceed the table's {self.width * self.page_size}")
            todo += [(slot, at) for at in range(ends.get(slot, self._end[slot]), end)]
            ends[slot] = max(end, ends.get(slot, 0))
        if len(todo) > len(self._free):
            raise RuntimeError(f"the page pool is exhausted: {len(todo)} pages needed, {len(self._free)} of {self.pages} free")
        for slot, at in todo:
            page = self._free.pop()
            self._uses[page] = 1
            self._set(slot, at, page)
            self._end[slot] = at + 1

    def trim(self, slot, first, keep=0):
        """Lets go of the pages that hold only positions below `first`, but for those of the first `keep`."""
        self._check(slot)
        end = min(int(first) // self.page_size, self._end[slot])
        begin = max(self._begin[slot], -(-int(keep) // self.page_size))
        for at in range(begin, end):
            self._drop(slot, at)
        self._begin[slot] = max(begin, end) if end > begin else self._begin[slot]

    def release(self, slot):
        """Lets go of all of the slot's pages."""
        self._check(slot)
        for at in range(self._end[slot]):
            self._drop(slot, at)
        self._end[slot] = self._begin[slot] = 0

    def share(self, slot, source, length):
        """Gives the (empty) slot the whole pages of the source's first `length` positions and, for what is left of them, a
        new page. Returns (page of the source, new page) when that is something, to be copied, else None. RuntimeError
        when the pool has no page for it, ValueError when the source has let go of one."""
        self._check(slot, source)
        whole, rest = divmod(max(int(length), 0), self.page_size)
        if self._end[slot]:
            raise ValueError(f"slot {slot} holds pages")
        if not self.has(source, length):
            raise ValueError(f"slot {source} does not hold its first {length} positions")
        if rest and not self._free:
            raise RuntimeError(f"the page pool is exhausted: 1 page needed, 0 of {self.pages} free")
        for at in range(whole):
            page = int(self._host[source, at])
            self._uses[page] += 1
            self._set(slot, at, page)
        self._end[slot] = whole
        if not rest:
            return None
        self.grow([(slot, length)])
        return int(self._host[source, whole]), int(self._host[slot, whole])

    @torch.inference_mode()
    def flush(self):
        """Sends the table's changes on the current stream."""
        while self._changed:
            if self._index is None:
                dev = self.table.device
                self._index = Upload(torch.zeros(self.SEND, dtype=torch.int64, device=dev))
                self._value = Upload(torch.zeros(self.SEND, dtype=torch.int32, device=dev))
            part = list(self._changed.items())[:self.SEND]
            n = len(part)
            self._index.buffer()[:n] = [at for at, _ in part]
            self._value.buffer()[:n] = [page for _, page in part]
            self._index.send(n)
            self._value.send(n)
            self.table.view(-1).index_copy_(0, self._index.dev[:n], self._value.dev[:n])
            for at, _ in part:
                del self._changed[at]
