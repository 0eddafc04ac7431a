"""A cache of pages for many sequences: which pages each sequence has, which of them are shared, which are free.

The keys and values are one buffer [layers, 2, pages, page_size, kv_heads, head_dim] that programs read through
`Builder.paged_attention` and that `Client.write_pages` / `Client.copy_pages` change in place; this class is the bookkeeping around it,
on the host. (The reference's example keeps one dense cache per layer for one sequence, examples/gemma/main.py:113-123.)
"""
from __future__ import annotations

import numpy as np

from . import INVALID_ARGUMENT, NOT_FOUND, RESOURCE_EXHAUSTED, B200Error


class PagedCache:
    """Sequences by number. A fork shares the pages of its parent; a page that is shared is copied before a token is written behind
    its last one. Every call that raises has changed nothing."""

    def __init__(self, client, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: str = "bf16"):
        if min(layers, pages, page_size, kv_heads, head_dim) < 1:
            raise B200Error("a cache has one layer, page, position, head and feature at least", INVALID_ARGUMENT)
        self.client, self.page_size, self.pages = client, page_size, pages
        self.shape = (layers, 2, pages, page_size, kv_heads, head_dim)
        self.buffer = self._zeros(dtype)
        self._free = list(range(pages - 1, -1, -1))            # the lowest number is taken first
        self._uses = [0] * pages
        self._pages: dict[int, list[int]] = {}
        self._lengths: dict[int, int] = {}
        self._next = 0

    def _zeros(self, dtype: str):
        from .shlo.builder import Builder
        b = Builder()
        return self.client.compile(b.module([b.full(self.shape, 0.0, dtype)])).execute([])[0]

    # ---- sequences ---------------------------------------------------------------
    def add(self) -> int:
        """A new empty sequence."""
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._lengths[seq] = [], 0
        return seq

    def fork(self, seq: int) -> int:
        """A new sequence with the tokens of another. No key or value is copied until one of the two grows."""
        pages = self._of(seq)
        new = self.add()
        self._pages[new], self._lengths[new] = list(pages), self._lengths[seq]
        for p in pages:
            self._uses[p] += 1
        return new

    def free(self, seq: int):
        """Ends a sequence; pages that nobody else has are free again."""
        for p in self._of(seq):
            self._uses[p] -= 1
            if self._uses[p] == 0:
                self._free.append(p)
        del self._pages[seq], self._lengths[seq]
        self._free.sort(reverse=True)

    def extend(self, seqs, counts) -> np.ndarray:
        """Room for counts[i] more tokens of sequence seqs[i], each sequence once: their slots for `write`, one sequence behind
        another. Shared last pages are copied first."""
        seqs, counts = [int(s) for s in seqs], [int(n) for n in counts]
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or any(n < 0 for n in counts):
            raise B200Error("extend takes each sequence once and a number of tokens for each", INVALID_ARGUMENT)
        size, need, copies = self.page_size, 0, []
        uses = {}
        for s, n in zip(seqs, counts):
            pages, length = self._of(s), self._lengths[s]
            if n and length % size:                            # the last page gets tokens behind those that it has
                last = pages[-1]
                if uses.setdefault(last, self._uses[last]) > 1:
                    uses[last] -= 1
                    copies.append(s)
            need += -(-(length + n) // size) - len(pages)
        if need + len(copies) > len(self._free):
            raise B200Error(f"{need + len(copies)} pages are needed and {len(self._free)} of {self.pages} are free", RESOURCE_EXHAUSTED)
        free, pairs, grown = list(self._free), [], {s: list(self._pages[s]) for s in seqs}
        for s in copies:
            pairs.append((grown[s][-1], free.pop()))
            grown[s][-1] = pairs[-1][1]
        slots = []
        for s, n in zip(seqs, counts):
            length = self._lengths[s]
            while len(grown[s]) * size < length + n:
                grown[s].append(free.pop())
            at = np.arange(length, length + n)
            slots.append(np.asarray(grown[s] or [0])[at // size] * size + at % size)
        if pairs:
            self.client.copy_pages(self.buffer, pairs)
        for s, n in zip(seqs, counts):
            for old, new in zip(self._pages[s], grown[s]):
                if old != new:
                    self._uses[old] -= 1
                    self._uses[new] = 1
            for new in grown[s][len(self._pages[s]):]:
                self._uses[new] = 1
            self._pages[s] = grown[s]
            self._lengths[s] += n
        self._free = free
        return np.concatenate(slots).astype(np.int32) if slots else np.zeros(0, np.int32)

    def write(self, rows, slots):
        """Keys and values [layers, 2, tokens, kv_heads, head_dim] of the tokens whose slots `extend` gave."""
        self.client.write_pages(self.buffer, rows, slots)

    def compact(self) -> int:
        """Moves the pages in use to the lowest numbers; gives how many moved. Tables and slots made before are void."""
        used = sorted({p for pages in self._pages.values() for p in pages})
        holes = [p for p in range(len(used)) if self._uses[p] == 0]
        moves = dict(zip([p for p in used if p >= len(used)], holes))
        if moves:
            self.client.copy_pages(self.buffer, list(moves.items()))
        for pages in self._pages.values():
            pages[:] = [moves.get(p, p) for p in pages]
        for old, new in moves.items():
            self._uses[new], self._uses[old] = self._uses[old], 0
        self._free = list(range(self.pages - 1, len(used) - 1, -1))
        return len(moves)

    # ---- what programs are given --------------------------------------------------
    def table(self, seqs, width: int | None = None) -> np.ndarray:
        """i32[sequences, width]: the pages of each, -1 behind the last. `width`: pages that a row has room for."""
        rows = [self._of(s) for s in seqs]
        most = max([len(r) for r in rows], default=0)
        width = most if width is None else width
        if most > width:
            raise B200Error(f"a sequence has {most} pages, the table has room for {width}", INVALID_ARGUMENT)
        out = np.full((len(rows), width), -1, np.int32)
        for i, r in enumerate(rows):
            out[i, :len(r)] = r
        return out

    def lengths(self, seqs) -> np.ndarray:
        """i32[sequences]: tokens of each."""
        for s in seqs:
            self._of(s)
        return np.asarray([self._lengths[s] for s in seqs], np.int32)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _of(self, seq: int) -> list[int]:
        if seq not in self._pages:
            raise B200Error(f"there is no sequence {seq}", NOT_FOUND)
        return self._pages[seq]
