"""Paged key/value cache of a model's attention layers, for ops.kv_append and
ops.paged_attention: one pool of pages per layer, one page table for all of them.

A sequence owns a list of pages; `fork` lets another sequence start from it with
the same pages (a prompt that is sampled several times is stored once), and a page
that several sequences hold is copied when one of them writes to it.  Pages lie
head by head in memory, (pages, heads, page size, head dim), so that a head's keys
of a page are one contiguous run; the tensors handed out are (pages, page size,
heads, head dim) views.  All bookkeeping is on the host and needs no
synchronisation; pools grow by doubling.
"""

from __future__ import annotations

import torch


def _ints(values, device):
    """int32 on the device; the copy is in stream order, from pinned memory that torch
    keeps until it is done."""
    t = torch.tensor(values, dtype=torch.int32, pin_memory=device.type == "cuda")
    return t.to(device, non_blocking=True)


class PagedStep(list):
    """The segments of one model step, with what the attention layers of the step
    share: positions, page table, offsets and lengths (int32, on the device) and
    the runs of keys that consecutive sequences have in common."""

    def __init__(self, cache, segments, positions):
        super().__init__(segments)
        self.cache = cache
        dev = cache.device
        self.positions = positions.to(torch.int32)
        self.longest = max((b - a for a, b, _, _ in segments), default=0)
        self.table, self.shared = cache.table([sid for _, _, sid, _ in segments])
        self.seq_lens = _ints([p0 + b - a for a, b, _, p0 in segments], dev)
        single = all(a == i and b == i + 1 for i, (a, b, _, _) in enumerate(segments))
        self.starts = None if single else _ints([segments[0][0]] + [b for _, b, _, _ in segments], dev)


class PagedKVCache:
    """layers x (keys, values) of `heads` heads of `head_dim`, in pages of `page_size`
    positions (a multiple of 16)."""

    def __init__(self, layers, heads, head_dim, page_size=64, device="cuda", dtype=torch.bfloat16):
        if page_size <= 0 or page_size % 16:
            raise ValueError(f"page_size must be a positive multiple of 16, got {page_size}")
        self.layers, self.heads, self.head_dim = layers, heads, head_dim
        self.page_size, self.device, self.dtype = page_size, torch.device(device), dtype
        self.clear()

    def clear(self):
        """Drops every sequence and the pools."""
        self._pools = [[None, None] for _ in range(self.layers)]
        self._free, self._holders, self._pages, self._lengths = [], [], {}, {}
        self._version, self._tables = 0, {}

    # ---- pages ----------------------------------------------------------------
    def _grow(self, pages):
        # One tensor after the other, each old one dropped before the next is made: the
        # old pools, what they grow by and one tensor are all that is held at a time.
        for pool in self._pools:
            for i in range(2):
                t = torch.empty(pages, self.heads, self.page_size, self.head_dim, dtype=self.dtype,
                                device=self.device)
                if pool[i] is not None:
                    t[:pool[i].shape[0]] = pool[i]
                pool[i] = t
        self._free += range(pages - 1, len(self._holders) - 1, -1)
        self._holders += [0] * (pages - len(self._holders))

    def _take(self):
        if not self._free:
            self._grow(max(16, 2 * len(self._holders)))
        page = self._free.pop()
        self._holders[page] = 1
        return page

    def _drop(self, page):
        self._holders[page] -= 1
        if self._holders[page] == 0:
            self._free.append(page)

    def layer(self, index):
        """(keys, values) of a layer: (pages, page size, heads, head dim)."""
        k, v = (t[:len(self._holders)] for t in self._pools[index])  # (more after a failed growth)
        return k.transpose(1, 2), v.transpose(1, 2)

    # ---- sequences ------------------------------------------------------------
    def extend(self, sid, start, end):
        """Pages for positions [start, end) of sequence `sid`, which this sequence alone
        may write; start 0 begins the sequence anew."""
        if start == 0:
            self.release(sid)
        length = self._lengths.get(sid, 0)
        if start > length:
            raise ValueError(f"sequence {sid} has {length} positions, cannot continue at {start}")
        pages = self._pages.setdefault(sid, [])
        for i in range(start // self.page_size, min(-(-end // self.page_size), len(pages))):
            if self._holders[pages[i]] > 1:  # copy on write
                new = self._take()
                for k, v in self._pools:
                    k[new], v[new] = k[pages[i]], v[pages[i]]
                self._drop(pages[i])
                pages[i] = new
                self._version += 1
        while len(pages) * self.page_size < end:
            pages.append(self._take())
            self._version += 1
        self._lengths[sid] = max(length, end)

    def fork(self, src, dst, length):
        """Sequence `dst` becomes the first `length` positions of `src`, on its pages."""
        if not 0 <= length <= self._lengths[src]:
            raise ValueError(f"sequence {src} has fewer than {length} positions")
        held = self._pages[src][:-(-length // self.page_size)]
        for page in held:
            self._holders[page] += 1
        self.release(dst)
        self._pages[dst], self._lengths[dst] = held, length
        self._version += 1

    def release(self, sid):
        self._lengths.pop(sid, None)
        for page in self._pages.pop(sid, ()):
            self._drop(page)
        self._version += 1

    # ---- what a step needs ------------------------------------------------------
    def step(self, segments, positions):
        """Room for the segments' new positions, and the step's PagedStep."""
        for a, b, sid, p0 in segments:
            self.extend(sid, p0, p0 + b - a)
        return PagedStep(self, segments, positions)

    def table(self, sids):
        """(page table (sequences, pages) int32, keyword arguments of paged_attention that
        describe the shared runs), rebuilt only when a page changed hands."""
        key = tuple(sids)
        hit = self._tables.get(key)
        if hit is not None and hit[0] == self._version:
            return hit[1]
        rows = [self._pages[s] for s in sids]
        width = max((len(r) for r in rows), default=0)
        table = _ints([r + [0] * (width - len(r)) for r in rows], self.device)
        made = table, self._shared(rows)
        self._tables = {key: (self._version, made)}
        return made

    def _shared(self, rows):
        """Consecutive sequences whose first pages are the same form a group; its run
        is the pages that all of them have."""
        starts, runs = [0], []
        for i, r in enumerate(rows):
            if i and r and rows[i - 1] and r[0] == rows[starts[-1]][0]:
                n = min(runs[-1], len(r))
                first = rows[starts[-1]]
                while first[:n] != r[:n]:
                    n -= 1
                runs[-1] = n
                continue
            if i:
                starts.append(i)
            runs.append(len(r))
        lens = [n * self.page_size if e - b > 1 else 0
                for n, b, e in zip(runs, starts, starts[1:] + [len(rows)])]
        if not any(lens):
            return {}
        return dict(shared_lens=_ints(lens, self.device), group_start=_ints(starts + [len(rows)], self.device))
