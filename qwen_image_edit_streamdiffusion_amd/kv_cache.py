"""Paged k / v cache of a decoder's layers: what a prompt's first tokens gave is kept in pages of
``page_size`` tokens, shared by the sequences that begin with them, and read by ``ops.attention_paged``.

The reference keeps whole prompt embeddings (README.md:124-125, cached_pipeline / VLM cache): a
changed instruction re-encodes the template and the picture before it. With the pages of a sequence
kept, ``fork`` starts the new one behind the tokens that both share.

Pages, lengths and tables live on the host (a few integers a sequence); ``step`` hands a forward over
new tokens its device arrays. k and v are [layers, pages, kv_heads, page_size, head_dim]: a page of one
kv head is one run of memory, as the attention's tiles read it. Pages are reused in the order of the
caller's stream: run a cache on one stream."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Sequence

import torch

from . import ops


class CacheFull(RuntimeError):
    """Too few free pages for the tokens of a step."""


@dataclass
class CacheStep:
    """Device arrays of one forward over new tokens (``PagedKVCache.step``)."""

    page_table: torch.Tensor  # int32 [seqs, width]
    kv_lens: torch.Tensor     # int32 [seqs], the new tokens included
    cu_seqlens: torch.Tensor  # int32 [seqs + 1] of the new tokens
    slots: torch.Tensor       # int64 [new tokens]


@dataclass
class _Sequence:
    pages: List[int]
    length: int


class PagedKVCache:
    def __init__(self, layers: int, kv_heads: int, head_dim: int, pages: int, page_size: int = 64, device="cuda"):
        if layers < 1 or kv_heads < 1 or pages < 1 or head_dim < 8 or head_dim % 8:
            raise ValueError("layers, kv_heads, pages >= 1 and head_dim a multiple of 8")
        if not (16 <= page_size <= 1024 and page_size & (page_size - 1) == 0):
            raise ValueError("page_size: a power of two in [16, 1024]")
        self.page_size, self.num_pages, self.device = page_size, pages, torch.device(device)
        self.k = torch.empty(layers, pages, kv_heads, page_size, head_dim, dtype=torch.bfloat16, device=device)
        self.v = torch.empty_like(self.k)
        self._free = list(range(pages - 1, -1, -1))
        self._users = [0] * pages  # sequences that hold a page
        self._seqs: Dict[int, _Sequence] = {}
        self._next = 0

    # ------------------------------------------------------------------ sequences
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        return self._seqs[seq].length

    def held_pages(self, seq: int) -> int:
        """Pages that hold a sequence's tokens, those that it shares among them."""
        return len(self._seqs[seq].pages)

    def add(self) -> int:
        """A new, empty sequence."""
        self._next += 1
        self._seqs[self._next] = _Sequence([], 0)
        return self._next

    def _take(self, n: int) -> List[int]:
        if n > len(self._free):
            raise CacheFull(f"{n} pages wanted, {len(self._free)} of {self.num_pages} free")
        got = [self._free.pop() for _ in range(n)]
        for p in got:
            self._users[p] = 1
        return got

    def _give(self, pages: Sequence[int]) -> None:
        for p in pages:
            self._users[p] -= 1
            if not self._users[p]:
                self._free.append(p)

    def fork(self, seq: int, length: int) -> int:
        """A new sequence that begins with the first ``length`` tokens of ``seq``: whole pages are
        shared, a page that ends behind them is copied."""
        src = self._seqs[seq]
        if not 0 <= length <= src.length:
            raise ValueError(f"{length} of {src.length} tokens")
        whole, rest = divmod(length, self.page_size)
        own = self._take(1) if rest else []
        if rest:
            try:
                for t in (self.k, self.v):
                    ops.copy_batched(t[:, src.pages[whole]], t[:, own[0]])
            except BaseException:
                self._give(own)
                raise
        for p in src.pages[:whole]:
            self._users[p] += 1
        new = self.add()
        self._seqs[new] = _Sequence(src.pages[:whole] + own, length)
        return new

    def drop(self, seq: int) -> None:
        """Give a sequence's pages back (shared ones when their last user goes)."""
        self._give(self._seqs.pop(seq).pages)

    # ------------------------------------------------------------------ a forward over new tokens
    def pages_needed(self, seq: int, new: int) -> int:
        s = self._seqs[seq]
        return -(-(s.length + new) // self.page_size) - len(s.pages)

    def step(self, seqs: Sequence[int], new: Sequence[int]) -> CacheStep:
        """Room for ``new[i]`` more tokens of each sequence, which are counted from here on: the forward
        that follows writes them (``ops.rope_append`` at ``slots``, layer by layer) before it reads them."""
        if len(seqs) != len(new) or not seqs or len(set(seqs)) != len(seqs) or any(n < 0 for n in new):
            raise ValueError("one count of new tokens for each of distinct sequences")
        need = [self.pages_needed(s, n) for s, n in zip(seqs, new)]
        if sum(need) > len(self._free):
            raise CacheFull(f"{sum(need)} pages wanted, {len(self._free)} of {self.num_pages} free")
        P, slots, lens, cu, table = self.page_size, [], [], [0], []
        free = iter(reversed(self._free))  # in the order in which _take gives them
        for seq, n, m in zip(seqs, new, need):
            s = self._seqs[seq]
            pages = s.pages + [next(free) for _ in range(m)]
            slots += [pages[i // P] * P + i % P for i in range(s.length, s.length + n)]
            lens.append(s.length + n)
            cu.append(cu[-1] + n)
            table.append(pages)
        width = max(1, max(map(len, table)))
        i32 = lambda v: torch.tensor(v, dtype=torch.int32).to(self.device)  # noqa: E731
        step = CacheStep(i32([t + [0] * (width - len(t)) for t in table]), i32(lens), i32(cu),
                         torch.tensor(slots, dtype=torch.int64).to(self.device))
        for seq, n, m in zip(seqs, new, need):  # the arrays are there: the tokens count
            s = self._seqs[seq]
            s.pages += self._take(m)
            s.length += n
        return step

    def take_back(self, seqs: Sequence[int], new: Sequence[int]) -> None:
        """Undo the last ``step`` of these sequences, as where its forward failed: the tokens are no longer
        counted, the pages that only they needed are free. Not once the sequences were forked behind it."""
        if len(seqs) != len(new) or len(set(seqs)) != len(seqs):
            raise ValueError("one count of tokens for each of distinct sequences")
        steps = [(self._seqs[seq], n) for seq, n in zip(seqs, new)]
        keep = [-(-(s.length - n) // self.page_size) for s, n in steps]
        if any(not 0 <= n <= s.length for s, n in steps):
            raise ValueError("more tokens than the sequence has")
        # the pages that hold such tokens, a part of the first one's slots may stay
        if any(self._users[p] != 1 for s, n in steps if n for p in s.pages[(s.length - n) // self.page_size:]):
            raise ValueError("pages that another sequence shares")
        for (s, n), k in zip(reversed(steps), reversed(keep)):  # the free pages in their order before the step
            self._free += reversed(s.pages[k:])
            for p in s.pages[k:]:
                self._users[p] = 0
            s.pages, s.length = s.pages[:k], s.length - n
