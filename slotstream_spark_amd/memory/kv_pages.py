"""Pages of a key-value cache and who holds them.

KVPages keeps the keys and values of `layers` attention layers in pages of `page` tokens (the layout that
kernels/paged_attention.py reads), hands pages to sequences, and keeps the device table that names them. Like the expert
pool's, its calls are host-side management: they run between launches or graph replays, on the current stream of the device,
and the kernels read the table they leave. A fork shares the pages of its source: each page counts its holders, and a page that
is to be written while others hold it is copied first. Moves of pages are one launch for all layers (ssmoe_move_pages).

No reference counterpart by interface (its caches are those of QSA, kernels/vendored.py:105-118); the error for too few pages is
the pool's Exhausted, and as there nothing changes when it is raised.
"""
from __future__ import annotations

import heapq

import numpy as np
import torch

from .. import _lib
from ..kernels.kv_pages import move_pages
from ..kernels.paged_attention import DIMS, PAGES, TYPES


class KVPages:
    """`n_pages` pages for `layers` layers: k [layers, n_pages, kv_heads, page, dim], v [layers, n_pages, kv_heads, dim,
    page], zero at first. Up to `max_seqs` sequences of up to `max_tokens` tokens; table int32 [max_seqs, width] on the device, -1
    where a sequence holds no page. `length[s]` is the number of tokens that a sequence has room for and counts as its own.
    `resizes` counts the times that k and v became other tensors (a captured graph holds the ones it was captured with). A page given
    back may be handed out at once: where sequences are worked on in several streams, their owners wait for each other first."""

    def __init__(self, layers: int, n_pages: int, kv_heads: int, dim: int, page: int = 64, max_seqs: int = 1,
                 max_tokens: int = 131072, dtype=torch.bfloat16, device="cuda"):
        if layers < 1 or n_pages < 1 or kv_heads < 1 or max_seqs < 1 or max_tokens < 1:
            raise ValueError("layers, n_pages, kv_heads, max_seqs and max_tokens must be positive")
        if page not in PAGES or dim not in DIMS or dtype not in TYPES:
            raise ValueError("pages hold 16, 32, 64, 128 or 256 tokens of 64, 128 or 256 bf16 or fp16 dimensions")
        self.layers, self.n_pages, self.kv_heads, self.dim, self.page = layers, n_pages, kv_heads, dim, page
        self.max_seqs, self.width = max_seqs, -(-max_tokens // page)
        self.k = torch.zeros((layers, n_pages, kv_heads, page, dim), dtype=dtype, device=device)
        self.v = torch.zeros((layers, n_pages, kv_heads, dim, page), dtype=dtype, device=device)
        self.table = torch.full((max_seqs, self.width), -1, dtype=torch.int32, device=device)
        self._table = np.full((max_seqs, self.width), -1, np.int32)
        self._refs = np.zeros(n_pages, np.int64)
        self._free = list(range(n_pages))   # a heap: the lowest id goes first
        self.length = [0] * max_seqs
        self.resizes = 0
        self._live = [False] * max_seqs

    # ------------------------------------------------------------------ what is held
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def pages_of(self, seq: int) -> list[int]:
        """The pages a sequence holds, in the order of its tokens (-1 where one was evicted)."""
        self._check(seq)
        return self._table[seq, :-(-self.length[seq] // self.page)].tolist()

    def _check(self, seq: int) -> None:
        if not 0 <= seq < self.max_seqs or not self._live[seq]:
            raise ValueError(f"no sequence {seq}")

    def _take(self, n: int) -> list[int]:
        if n > len(self._free):
            raise _lib.Exhausted(f"{n} pages are needed, {len(self._free)} of {self.n_pages} are free")
        ids = [heapq.heappop(self._free) for _ in range(n)]
        self._refs[ids] = 1
        return ids

    def _drop(self, ids) -> None:
        for p in ids:
            if p >= 0:
                self._refs[p] -= 1
                if self._refs[p] == 0:
                    heapq.heappush(self._free, int(p))

    def _publish(self, seq: int) -> None:
        self.table[seq].copy_(torch.from_numpy(self._table[seq]))

    def _move(self, src, dst, table=None) -> None:
        move_pages(self.k, self.v, torch.tensor(src, dtype=torch.int32).to(self.k.device),
                   torch.tensor(dst, dtype=torch.int32).to(self.k.device), table)

    # ------------------------------------------------------------------ sequences
    def new(self) -> int:
        """An empty sequence."""
        for s in range(self.max_seqs):
            if not self._live[s]:
                self._live[s], self.length[s] = True, 0
                return s
        raise _lib.Exhausted(f"all {self.max_seqs} sequences are in use")

    def extend(self, seq: int, tokens: int) -> None:
        """Room for `tokens` more tokens, which count as the sequence's own from now on. Pages of them that other sequences
        hold too are copied first."""
        self._check(seq)
        if tokens < 0:
            raise ValueError(f"cannot extend by {tokens} tokens; truncate() takes tokens away")
        self.rewrite(seq, self.length[seq], tokens)

    def rewrite(self, seq: int, at: int, tokens: int) -> None:
        """truncate() to `at` and extend() by `tokens` in one: pages that both have stay, those given up serve the same call, and
        where it is refused the sequence keeps what it had."""
        self._check(seq)
        if not 0 <= at <= self.length[seq] or tokens < 0:
            raise ValueError(f"cannot write {tokens} tokens from {at} on over {self.length[seq]}")
        want = at + tokens
        if want > self.width * self.page:
            raise ValueError(f"{want} tokens exceed the table's {self.width * self.page}")
        row, last = self._table[seq], -(-want // self.page)
        first = at // self.page if tokens else last
        new = [w for w in range(first, last) if row[w] < 0 or self._refs[row[w]] > 1]
        kept = int(row[first]) if at % self.page and first in new else None   # holds tokens before `at`
        if kept == -1:
            raise ValueError(f"the page of token {at - 1} of sequence {seq} was evicted")
        gone = row[last:][row[last:] >= 0].tolist()
        if len(new) > self.free_pages + sum(self._refs[p] == 1 for p in gone):
            self._take(len(new))   # raises: nothing has changed yet
        self._drop(gone)
        row[last:] = -1
        ids = self._take(len(new))
        if kept is not None:
            self._move([kept], ids[:1])
        self._drop(row[new].tolist())
        row[new] = ids
        self.length[seq] = want
        if ids or gone:
            self._publish(seq)

    def reserve(self, seq: int, tokens: int) -> None:
        """extend() up to `tokens` tokens in all, where there are fewer."""
        self._check(seq)
        if tokens > self.length[seq]:
            self.extend(seq, tokens - self.length[seq])

    def truncate(self, seq: int, length: int) -> None:
        """Keeps the first `length` tokens and gives back the pages past them."""
        self._check(seq)
        if not 0 <= length <= self.length[seq]:
            raise ValueError(f"cannot keep {length} of {self.length[seq]} tokens")
        self.rewrite(seq, length, 0)

    def free(self, seq: int) -> None:
        """Gives back every page of a sequence and the sequence itself."""
        self.truncate(seq, 0)
        self._live[seq] = False

    def fork(self, seq: int) -> int:
        """A new sequence with the same tokens: it shares the full pages; the last page, where it has room left, is copied."""
        self._check(seq)
        child = self.new()
        row, n = self._table[seq], self.length[seq]
        try:
            own = self._take(1) if n % self.page and row[n // self.page] >= 0 else []
        except _lib.Exhausted:
            self._live[child] = False
            raise
        held = -(-n // self.page)
        mine = self._table[child]
        mine[:held] = row[:held]
        if own:
            self._move([int(row[held - 1])], own)
            mine[held - 1] = own[0]
        for p in mine[:held - 1 if own else held]:
            if p >= 0:
                self._refs[p] += 1
        self.length[child] = n
        self._publish(child)
        return child

    def evict(self, seq: int, window: int, sinks: int = 0, back: int = 8) -> int:
        """Gives back the pages that no row from `back` tokens before the end on sees under a window of `window` tokens with
        `sinks` first ones kept (`back`: how many tokens may still be truncated). Returns their number."""
        self._check(seq)
        if window < 1 or sinks < 0 or back < 0:
            raise ValueError("need window >= 1, sinks >= 0 and back >= 0")
        first = max(0, self.length[seq] - back - window + 1) // self.page
        kept = -(-sinks // self.page)
        row = self._table[seq]
        gone = [w for w in range(kept, first) if row[w] >= 0]
        if gone:
            self._drop(row[gone].tolist())
            row[gone] = -1
            self._publish(seq)
        return len(gone)

    # ------------------------------------------------------------------ the pool
    def compact(self) -> int:
        """Moves the held pages to the lowest ids (the tables follow on the device, in the same launch) and returns how many
        pages are held."""
        held = np.flatnonzero(self._refs)
        n = len(held)
        src = held[held >= n]
        if len(src):
            dst = np.flatnonzero(self._refs[:n] == 0)
            self._move(src.tolist(), dst.tolist(), self.table)
            to = np.arange(self.n_pages, dtype=np.int32)
            to[src] = dst
            self._table = np.where(self._table >= 0, to[np.maximum(self._table, 0)], -1).astype(np.int32)
            self._refs[dst] = self._refs[src]
            self._refs[src] = 0
            self._free = np.flatnonzero(self._refs == 0).tolist()
        return n

    def resize(self, n_pages: int) -> None:
        """Another number of pages; fewer only down to those held (which are compacted first). k and v become other tensors."""
        if n_pages < 1:
            raise ValueError("need n_pages >= 1")
        held = int((self._refs > 0).sum())
        if n_pages < held:
            raise _lib.Exhausted(f"{held} pages are held, {n_pages} are asked for")
        if n_pages < self.n_pages:
            self.compact()
        keep = min(n_pages, self.n_pages)

        def sized(t):
            out = torch.zeros((self.layers, n_pages, *t.shape[2:]), dtype=t.dtype, device=t.device)
            out[:, :keep] = t[:, :keep]
            return out

        self.k, self.v = sized(self.k), sized(self.v)
        self.resizes += 1
        refs = np.zeros(n_pages, np.int64)
        refs[:keep] = self._refs[:keep]
        self._refs, self.n_pages = refs, n_pages
        self._free = np.flatnonzero(refs == 0).tolist()
