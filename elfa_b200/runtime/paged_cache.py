"""The key / value cache of many sequences in pages: who has which page, and what the kernels of :mod:`elfa_b200.ops.paged` need to know of a call.

One pool ``[layers, pages, 2, kv_heads, page, head_dim]``; a sequence is a list of page numbers that holds in all layers. Sequences that fork share their pages until one of
them writes; with a window, pages that no later token can see go back; compacting moves the pages in use to the front. Page numbers are the host's business
(nothing here waits for the device), what they name is moved by kernels on the current stream: use one cache from one stream at a time.

reference: ``src/eval/evaluator.zig:419-470`` (no cache: every token runs the whole context of one sequence again).
"""
from __future__ import annotations

import heapq
from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence

import torch

from .. import ops


class OutOfPages(RuntimeError):
    """The pool has fewer free pages than a call needs; nothing has changed."""


@dataclass
class PagedBatch:
    """One call's new tokens: those of sequence ``i`` are rows ``q_start[i]`` to ``q_start[i + 1]`` (see :mod:`elfa_b200.ops.paged`)."""
    table: torch.Tensor
    q_start: torch.Tensor
    kv_len: torch.Tensor
    positions: torch.Tensor          # [T] int64, of every new token in its sequence
    last: torch.Tensor               # [B] int64, the row of each sequence's last new token
    max_new: int
    end: int                         # one more than the largest position


@dataclass
class _Sequence:
    pages: List[int]                 # -1: no longer there
    length: int = 0
    kept: int = 0                    # pages before this one, but for the sinks, have gone back


class PagedCache:
    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16, device=None,
                 window: Optional[int] = None, sinks: int = 0):
        """``window``: tokens see the last ``window`` ones and the first ``sinks`` only, and pages that lie wholly between the two are given back."""
        if page_size not in ops.PAGE_SIZES:
            raise ValueError(f"page_size must be one of {ops.PAGE_SIZES}, got {page_size}")
        if layers < 1 or pages < 1 or (window is not None and window < 1) or sinks < 0:
            raise ValueError("a cache has layers and pages, a window holds at least the token itself, and there are no negative sinks")
        if torch.empty(0, device=device).is_cuda and (dtype is not torch.bfloat16 or head_dim % 8 or not 8 <= head_dim <= 128):
            raise ValueError(f"a cache on the device holds bf16 and head dimensions that are multiples of 8 up to 128, got {dtype} and {head_dim}")
        self.pool = torch.zeros((layers, pages, 2, kv_heads, page_size, head_dim), dtype=dtype, device=device)
        self.page_size, self.window, self.sinks = page_size, window, sinks
        self._refs = [0] * pages
        self._free = list(range(pages))                          # a heap: the lowest number first
        self._seqs: Dict[int, _Sequence] = {}
        self._next = 0

    # ------------------------------------------------------------------------------------------------ sequences
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        return self._seqs[seq].length

    def pages_of(self, seq: int) -> List[int]:
        return list(self._seqs[seq].pages)

    def add(self) -> int:
        """An empty sequence."""
        self._seqs[self._next] = _Sequence([])
        self._next += 1
        return self._next - 1

    def fork(self, seq: int, n: int = 1) -> List[int]:
        """``n`` sequences with the tokens of ``seq``, on the same pages."""
        s, out = self._seqs[seq], []
        for _ in range(n):
            for p in s.pages:
                if p >= 0:
                    self._refs[p] += 1
            self._seqs[self._next] = _Sequence(list(s.pages), s.length, s.kept)
            out.append(self._next)
            self._next += 1
        return out

    def free(self, seq: int) -> None:
        for p in self._seqs.pop(seq).pages:
            self._release(p)

    def _release(self, page: int) -> None:
        if page < 0:
            return
        self._refs[page] -= 1
        if self._refs[page] == 0:
            heapq.heappush(self._free, page)

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self._refs[page] = 1
        return page

    # ------------------------------------------------------------------------------------------------ a call
    def append(self, seqs: Sequence[int], new: Sequence[int]) -> PagedBatch:
        """Makes room for ``new[i]`` more tokens of ``seqs[i]``; their keys and values are written by the layers. A page that a sequence shares and would write
        to is copied first, in all layers by one launch. Raises :class:`OutOfPages` when the pool has not enough free pages, without a change."""
        if len(seqs) != len(new) or len(set(seqs)) != len(seqs) or not seqs:
            raise ValueError("as many numbers of tokens as sequences, at least one, each sequence once")
        if min(new) < 0:
            raise ValueError("a negative number of new tokens")
        if sum(new) == 0:
            raise ValueError("no new token")
        page = self.page_size
        need, shared = 0, {}
        for i, n in zip(seqs, new):
            s = self._seqs[i]
            need += -(-(s.length + n) // page) - len(s.pages)
            if n and s.length % page:
                last = s.pages[-1]
                # of the sequences that write to one page in this call and of all that hold it, the last one that is left may keep it
                shared[last] = shared.get(last, 0) + 1
                if self._refs[last] - shared[last] > 0:
                    need += 1
        if need > len(self._free):
            raise OutOfPages(f"{need} pages wanted, {len(self._free)} free")
        src, dst = [], []
        for i, n in zip(seqs, new):
            s = self._seqs[i]
            if n and s.length % page and self._refs[s.pages[-1]] > 1:
                self._refs[s.pages[-1]] -= 1
                src.append(s.pages[-1])
                s.pages[-1] = self._take()
                dst.append(s.pages[-1])
            for _ in range(-(-(s.length + n) // page) - len(s.pages)):
                s.pages.append(self._take())
            s.length += n
        ops.copy_pages(self.pool, src, dst)
        batch = self._batch(seqs, new)
        if self.window is not None:
            for i in seqs:
                self._trim(self._seqs[i])
        return batch

    def _batch(self, seqs: Sequence[int], new: Sequence[int]) -> PagedBatch:
        """All numbers of the call in one transfer."""
        B, T, N = len(seqs), sum(new), max(1, max(len(self._seqs[i].pages) for i in seqs))
        flat = torch.full((2 * B + 1 + B * N,), -1, dtype=torch.int32)
        start, lens, table = flat[:B + 1], flat[B + 1:2 * B + 1], flat[2 * B + 1:].view(B, N)
        at, pos = 0, torch.empty(T + B, dtype=torch.int64)
        start[0] = 0
        for j, (i, n) in enumerate(zip(seqs, new)):
            s = self._seqs[i]
            pos[at:at + n] = torch.arange(s.length - n, s.length)
            at += n
            start[j + 1], lens[j] = at, s.length
            pos[T + j] = at - 1
            if s.pages:
                table[j, :len(s.pages)] = torch.tensor(s.pages, dtype=torch.int32)
        dev = self.pool.device
        if dev.type == "cuda":                                   # from pageable memory: staged before the call returns, so the host's copy may go
            flat, pos = flat.to(dev, non_blocking=True), pos.to(dev, non_blocking=True)
            start, lens, table = flat[:B + 1], flat[B + 1:2 * B + 1], flat[2 * B + 1:].view(B, N)
        return PagedBatch(table, start, lens, pos[:T], pos[T:], max(new), max(self._seqs[i].length for i in seqs))

    def _trim(self, s: _Sequence) -> None:
        """Gives back the pages that the next token, and so any later one, does not see. The call under way still reads them: it comes first on the stream."""
        first = max(0, s.length - self.window + 1)               # first key of the next token's window
        keep = -(-self.sinks // self.page_size)                  # pages with sinks
        for p in range(max(s.kept, keep), min(first // self.page_size, len(s.pages))):
            self._release(s.pages[p])
            s.pages[p] = -1
        s.kept = max(s.kept, min(first // self.page_size, len(s.pages)))

    # ------------------------------------------------------------------------------------------------ layers
    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, batch: PagedBatch) -> None:
        ops.paged_write(k, v, self.pool[layer], batch.table, batch.q_start, batch.kv_len)

    def attend(self, layer: int, q: torch.Tensor, batch: PagedBatch) -> torch.Tensor:
        return ops.paged_attention(q, self.pool[layer], batch.table, batch.q_start, batch.kv_len, max_new=batch.max_new, window=self.window, sinks=self.sinks)

    # ------------------------------------------------------------------------------------------------ the pool
    def compact(self) -> int:
        """Moves the pages in use to the front of the pool; returns how many there are. Batches made before name the old places: make new ones."""
        used = [p for p, r in enumerate(self._refs) if r]
        n = len(used)
        src = [p for p in used if p >= n]
        dst = [p for p in range(n) if not self._refs[p]]
        ops.copy_pages(self.pool, src, dst)
        to = dict(zip(src, dst))
        for s in self._seqs.values():
            s.pages = [to.get(p, p) for p in s.pages]
        for a, b in to.items():
            self._refs[a], self._refs[b] = 0, self._refs[a]
        self._free = list(range(n, len(self._refs)))
        return n
