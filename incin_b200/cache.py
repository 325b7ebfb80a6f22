"""A paged key-value cache: the pages of all layers, and which sequence owns which.

A :class:`PagedCache` holds fixed pages of ``page_size`` tokens for every layer in one tensor and hands them out to sequences.
Sequences grow (:meth:`extend`), share their pages until one of them writes (:meth:`fork`), give pages back
(:meth:`truncate`, :meth:`free`) and can be moved to the front of the tensor (:meth:`compact`).  The bookkeeping is on the host,
where the lengths are known anyway; only page contents move on the device (``F.copy_pages``)::

    cache = PagedCache.of(model, pages=4096)
    a = cache.new()
    logits = model.extend(prompt, cache, [a], [len(prompt)])       # fills the cache, logits of the last token
    b = cache.fork(a)                                              # shares all pages
    logits = model.extend(next_tokens, cache, [a, b])              # one token each; the open page is copied first

All launches that touch one cache belong on one stream (or are ordered by events).
"""
from __future__ import annotations

import heapq
from collections import Counter
from contextlib import contextmanager
from dataclasses import dataclass, field

import torch

from .ops import functional as F
from .ops.paged import PAGE_SIZES, check_kernels


class CacheFull(RuntimeError):
    """The cache has too few free pages; nothing was changed."""


@dataclass
class _Sequence:
    pages: list[int] = field(default_factory=list)
    length: int = 0


class PagedBatch:
    """What one forward pass needs to know about its sequences, on the device (made by :meth:`PagedCache.extend`)."""

    def __init__(self, cache: "PagedCache", table: list[list[int]], lengths: list[int], counts: list[int]):
        width = max(1, max(len(t) for t in table))
        S = len(lengths)
        offsets = [0]
        for n in counts:
            offsets.append(offsets[-1] + n)
        flat = torch.tensor([p for t in table for p in t + [-1] * (width - len(t))] + lengths + offsets, dtype=torch.int32)
        flat = flat.to(cache.storage.device)
        self.cache = cache
        self.counts = counts
        self.rows = offsets[-1]
        self.starts = [n - c for n, c in zip(lengths, counts)]   # position of each sequence's first new token
        self.table = flat[:S * width].view(S, width)
        self.lengths = flat[S * width:S * width + S]
        self.offsets = flat[S * width + S:]
        self.single = all(n == 1 for n in counts)
        self._undo: list[tuple] = []     # what PagedCache.take_back needs

    def positions(self) -> torch.Tensor:
        """Positions of the new tokens, ``[rows]`` int64."""
        return torch.cat([torch.arange(a, a + n) for a, n in zip(self.starts, self.counts)]).to(self.table.device)

    def last_rows(self) -> torch.Tensor:
        """Row of each sequence's last new token, ``[sequences]`` int64."""
        return self.offsets[1:].long() - 1

    def attend(self, layer: int, qkv: torch.Tensor, n_heads: int, theta: float | None = None, scale: float | None = None) -> torch.Tensor:
        """The new tokens' keys and values enter layer ``layer``, their queries attend to it; ``qkv`` ``[rows, width]`` ->
        ``[rows, n_heads * head_dim]``."""
        k, v = self.cache.layer(layer)
        offsets = None if self.single else self.offsets
        q = F.kv_append(qkv, k, v, self.table, self.lengths, offsets, n_heads=n_heads, theta=theta)
        if self.single:
            return F.decode_attention(q, k, v, self.table, self.lengths, scale=scale).flatten(1)
        return F.prompt_attention(q, k, v, self.table, self.lengths, offsets, scale=scale).flatten(1)


class PagedCache:
    def __init__(self, n_layer: int, n_kv_head: int, head_dim: int, pages: int, *, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if min(n_layer, n_kv_head, head_dim, pages) <= 0:
            raise ValueError(f"layers, heads, head_dim and pages must be positive, got {n_layer}, {n_kv_head}, {head_dim}, {pages}")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        self.page_size = page_size
        self.n_pages = pages
        # [layer, key / value, page, head, token, element]: a page of one layer is one run of memory, a head's part another
        self.storage = torch.empty(n_layer, 2, pages, n_kv_head, page_size, head_dim, dtype=dtype, device=device)
        self._refs = [0] * pages
        self._free = list(range(pages))   # a heap: the lowest free page is taken first
        self._seqs: dict[int, _Sequence] = {}
        self._next = 0

    @classmethod
    def of(cls, model, pages: int, *, page_size: int = 64) -> "PagedCache":
        """A cache for ``model`` (``models.Llama`` or ``models.GPT2``), in its parameters' type and on their device.  Refused where
        the operators have no kernels for it: on CUDA they take bf16 and fp16 with head_dim 64 or 128."""
        cfg, p = model.cfg, next(model.parameters())
        heads = getattr(cfg, "n_kv_head", cfg.n_head)
        head_dim = getattr(cfg, "head_dim", cfg.d_model // cfg.n_head)
        if p.is_cuda:
            check_kernels("PagedCache", p.dtype, head_dim, cfg.n_head // heads)
        return cls(cfg.n_layer, heads, head_dim, pages, page_size=page_size, dtype=p.dtype, device=p.device)

    # ------------------------------------------------------------------------------------------------ what is in it
    def layer(self, i: int) -> tuple[torch.Tensor, torch.Tensor]:
        return self.storage[i, 0], self.storage[i, 1]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        return self._of(seq).length

    def pages_of(self, seq: int) -> list[int]:
        return list(self._of(seq).pages)

    def _of(self, seq: int) -> _Sequence:
        try:
            return self._seqs[seq]
        except KeyError:
            raise KeyError(f"no sequence {seq} in this cache") from None

    # ------------------------------------------------------------------------------------------------ sequences
    def _add(self, sequence: _Sequence) -> int:
        seq, self._next = self._next, self._next + 1
        self._seqs[seq] = sequence
        return seq

    def new(self) -> int:
        """A sequence without tokens; its handle is never given out again."""
        return self._add(_Sequence())

    def fork(self, seq: int) -> int:
        """A second sequence with the same tokens.  All pages are shared; the open one is copied when either side grows."""
        old = self._of(seq)
        for p in old.pages:
            self._refs[p] += 1
        return self._add(_Sequence(list(old.pages), old.length))

    def _drop(self, page: int) -> None:
        self._refs[page] -= 1
        if self._refs[page] == 0:
            heapq.heappush(self._free, page)

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self._refs[page] = 1
        return page

    def truncate(self, seq: int, length: int) -> None:
        """Forget the tokens of ``seq`` from position ``length`` on."""
        s = self._of(seq)
        if not 0 <= length <= s.length:
            raise ValueError(f"sequence {seq} has {s.length} tokens, cannot keep {length}")
        keep = -(-length // self.page_size)
        for p in s.pages[keep:]:
            self._drop(p)
        del s.pages[keep:]
        s.length = length

    def free(self, seq: int) -> None:
        """Give all pages of ``seq`` back and forget it."""
        self.truncate(seq, 0)
        del self._seqs[seq]

    def extend(self, seqs: list[int], counts: list[int] | None = None) -> PagedBatch:
        """Make room for ``counts[i]`` (default 1) new tokens of each sequence and describe the batch to the operators.
        A shared open page that is about to be written is copied first (all layers and all such pages in one launch).
        Raises :class:`CacheFull` when there are too few free pages; whatever it raises, nothing was changed.  The new tokens
        count as cached from here on: if what should write them fails, :meth:`take_back` the batch."""
        counts = [1] * len(seqs) if counts is None else [int(n) for n in counts]
        if not seqs or len(counts) != len(seqs) or len(set(seqs)) != len(seqs) or min(counts) < 0:
            raise ValueError(f"extend: sequences must be distinct, with one count >= 0 each, got {seqs} and {counts}")
        held = [self._of(s) for s in seqs]
        size = self.page_size
        need, leaving = 0, Counter()
        split = []   # whether a sequence's open page has to be copied
        for s, n in zip(held, counts):
            need += -(-(s.length + n) // size) - len(s.pages)
            page = s.pages[-1] if n and s.length % size else None
            shared = page is not None and self._refs[page] - leaving[page] > 1
            if shared:
                leaving[page] += 1
                need += 1
            split.append(shared)
        if need > len(self._free):
            raise CacheFull(f"{need} pages wanted, {len(self._free)} free of {self.n_pages}")
        src, dst, undo = [], [], []
        try:
            for s, n, copy in zip(held, counts, split):
                undo.append((s, s.length, len(s.pages), s.pages[-1] if copy else None))
                if copy:
                    old, s.pages[-1] = s.pages[-1], self._take()
                    self._refs[old] -= 1      # its other owners keep it
                    src.append(old)
                    dst.append(s.pages[-1])
                s.length += n
                while len(s.pages) * size < s.length:
                    s.pages.append(self._take())
            if src:
                self._copy(src, dst)
            batch = PagedBatch(self, [s.pages for s in held], [s.length for s in held], counts)
        except BaseException:
            self._restore(undo)
            raise
        batch._undo = undo
        return batch

    def _restore(self, undo: list[tuple]) -> None:
        while undo:
            s, length, pages, copied = undo.pop()
            for p in s.pages[pages:]:
                self._drop(p)
            del s.pages[pages:]
            if copied is not None and s.pages[-1] != copied:
                self._drop(s.pages[-1])
                s.pages[-1] = copied
                self._refs[copied] += 1
            s.length = length

    def take_back(self, batch: PagedBatch) -> None:
        """Undo the :meth:`extend` that made ``batch``: lengths, pages and their owners are as before it.  For a pass that failed,
        before anything else is done to the cache."""
        self._restore(batch._undo)

    def admit(self, tokens: torch.Tensor, seqs: list[int], counts: list[int] | None, max_seq: int) -> PagedBatch:
        """:meth:`extend` for a model's forward pass: ``tokens`` are the new tokens, no sequence may pass ``max_seq`` and
        every one gets a token at least (it has a last row)."""
        counts = [1] * len(seqs) if counts is None else list(counts)
        if tokens.dim() != 1 or tokens.shape[0] != sum(counts):
            raise ValueError(f"{tuple(tokens.shape)} tokens for counts {counts}")
        for s, n in zip(seqs, counts):
            if n < 1 or self.length(s) + n > max_seq:
                raise ValueError(f"sequence {s}: {n} new tokens after {self.length(s)}, the model holds {max_seq}")
        return self.extend(seqs, counts)

    @contextmanager
    def step(self, tokens: torch.Tensor, seqs: list[int], counts: list[int] | None, max_seq: int):
        """The batch of :meth:`admit` for a ``with`` block that runs the forward pass; an exception in it takes the tokens back."""
        batch = self.admit(tokens, seqs, counts, max_seq)
        try:
            yield batch
        except BaseException:
            self.take_back(batch)
            raise

    # ------------------------------------------------------------------------------------------------ pages
    def _copy(self, src: list[int], dst: list[int]) -> None:
        pairs = torch.tensor([src, dst], dtype=torch.int32).to(self.storage.device)
        F.copy_pages(self.storage, pairs[0], pairs[1])

    def compact(self) -> int:
        """Move the pages in use to the front of the storage; returns their number.  Batches made before hold old tables."""
        used = [p for p in range(self.n_pages) if self._refs[p]]
        n = len(used)
        src = [p for p in used if p >= n]
        dst = [p for p in range(n) if not self._refs[p]]
        if src:
            self._copy(src, dst)
            to = dict(zip(src, dst))
            for s in self._seqs.values():
                s.pages = [to.get(p, p) for p in s.pages]
            for a, b in to.items():
                self._refs[b], self._refs[a] = self._refs[a], 0
            self._free = list(range(n, self.n_pages))
        return n
