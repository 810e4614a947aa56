"""Paged key/value cache of many sequences of different lengths, joined and
retired while others run (no counterpart in the reference, whose KVCache holds
one sequence, src/model/chassis.py:262-330)."""
from __future__ import annotations

from typing import List, Sequence

import numpy as np
import torch

from .. import ops


class PagedKVCache:
    """``n_pages`` pages of ``page_size`` tokens per layer, [n_pages, n_head,
    page_size, head_dim], shared by up to ``max_seqs`` sequences of up to
    ``max_seq_len`` tokens.

        cache = PagedKVCache(n_layers, 512, 64, n_head, head_dim, device, dtype)
        a, b = cache.add(2)
        batch = cache.select([a])
        logits, _ = model(prompt_a, kv_cache=batch); batch.increment(T)
        batch = cache.select([a, b])            # sequences of any lengths
        logits, _ = model(next_tokens, kv_cache=batch); batch.increment(1)
        cache.remove([b])                       # its pages are free again

    ``window`` > 0: a token sees the last ``window`` tokens and the first
    ``sinks``; pages behind the window are freed as the sequences grow.  Every
    call's tokens must be of one length per sequence (as any forward's)."""

    def __init__(self, n_layers: int, n_pages: int, page_size: int, n_head: int, head_dim: int, device,
                 dtype: torch.dtype = torch.float16, max_seqs: int = 64, max_seq_len: int = 4096, window: int = 0,
                 sinks: int = 0):
        if n_pages < 1 or page_size < 1 or max_seqs < 1 or max_seq_len < 1 or window < 0 or sinks < 0:
            raise ValueError("a paged cache needs pages, a page size, sequences and a length, and no negative window")
        self.n_layers, self.n_pages, self.page_size = n_layers, n_pages, page_size
        self.n_head, self.head_dim, self.dtype = n_head, head_dim, dtype
        self.max_seq_len, self.window, self.sinks = max_seq_len, window, sinks
        shape = (n_pages, n_head, page_size, head_dim)
        self.k_pages: List[torch.Tensor] = [torch.zeros(shape, device=device, dtype=dtype) for _ in range(n_layers)]
        self.v_pages: List[torch.Tensor] = [torch.zeros(shape, device=device, dtype=dtype) for _ in range(n_layers)]
        self.err = torch.zeros(1, dtype=torch.int32, device=device)
        self.device = self.err.device  # with its index: "cuda" may be another one by the next call
        self._free = list(range(n_pages - 1, -1, -1))
        self._rows = list(range(max_seqs - 1, -1, -1))
        self._table = np.full((max_seqs, -(-max_seq_len // page_size)), -1, dtype=np.int32)
        self._len = np.zeros(max_seqs, dtype=np.int64)
        self._used = np.zeros(max_seqs, dtype=bool)
        self._removed = np.zeros(max_seqs, dtype=np.int64)  # sequences removed from each row, which add() hands out again

    def add(self, n: int = 1) -> List[int]:
        """``n`` new empty sequences."""
        if n > len(self._rows):
            raise RuntimeError(f"{n} new sequences, but only {len(self._rows)} of {len(self._len)} are free")
        ids = [self._rows.pop() for _ in range(n)]
        self._used[ids] = True
        self._len[ids] = 0
        return ids

    def remove(self, seqs: Sequence[int]):
        """Frees the sequences and their pages."""
        for s in self._ids(seqs):
            row = self._table[s]
            self._free.extend(int(p) for p in row[row >= 0])
            row[:] = -1
            self._used[s] = False
            self._removed[s] += 1
            self._rows.append(int(s))

    def lengths(self, seqs: Sequence[int]) -> List[int]:
        return [int(n) for n in self._len[self._ids(seqs)]]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def select(self, seqs: Sequence[int]) -> "PagedBatch":
        """The given sequences, in this order, as a forward's ``kv_cache``."""
        return PagedBatch(self, self._ids(seqs))

    def check(self):
        """Raise if a kernel met a slot, page or length out of range since the last check (synchronises)."""
        if int(self.err.item()) != 0:
            self.err.zero_()
            raise IndexError("a paged-cache kernel met an index out of range")

    # -- bookkeeping ----------------------------------------------------------------
    def _ids(self, seqs) -> np.ndarray:
        ids = np.asarray(list(seqs), dtype=np.int64)
        if ids.ndim != 1 or len(set(ids.tolist())) != len(ids):
            raise ValueError(f"sequences must be distinct, got {seqs}")
        if len(ids) and (ids.min() < 0 or ids.max() >= len(self._len) or not self._used[ids].all()):
            raise ValueError(f"not all of {seqs} are sequences of this cache")
        return ids

    def _reserve(self, ids: np.ndarray, n: int):
        """Pages for ``n`` more tokens of each sequence; all or none."""
        new = self._len[ids] + n
        if len(ids) and int(new.max()) > self.max_seq_len:
            raise ValueError(f"a sequence of {int(new.max())} tokens, but the cache holds {self.max_seq_len} per sequence")
        ps = self.page_size
        want = [(s, p) for s, a, b in zip(ids, self._len[ids] // ps, -(-new // ps)) for p in range(a, b)
                if self._table[s, p] < 0]
        if len(want) > len(self._free):
            raise RuntimeError(f"KV cache is out of pages: {len(want)} wanted, {len(self._free)} free")
        for s, p in want:
            self._table[s, p] = self._free.pop()

    def _advance(self, ids: np.ndarray, n: int):
        self._len[ids] += n
        if not self.window:
            return
        ps = self.page_size
        first = -(-self.sinks // ps)                       # pages that hold sinks stay
        for s in ids:                                      # the next token sees keys from len - window + 1 on
            dead = self._table[s, first:max(first, (int(self._len[s]) - self.window + 1) // ps)]
            self._free.extend(int(p) for p in dead[dead >= 0])
            dead[:] = -1


class PagedBatch:
    """Some sequences of a PagedKVCache for one or more forwards."""

    def __init__(self, cache: PagedKVCache, ids: np.ndarray):
        self.cache, self.ids = cache, ids
        self.batch_size, self.dtype = len(ids), cache.dtype
        self._removed = cache._removed[ids]

    @property
    def longest(self) -> int:
        return int(self.cache._len[self.ids].max(initial=0))

    def _check(self):
        if (self.cache._removed[self.ids] != self._removed).any():
            raise ValueError("some of the batch's sequences were removed since it was selected")

    def increment(self, n: int = 1):
        """Counts the ``n`` tokens per sequence that the last forward stored."""
        if n < 0:
            raise ValueError(f"stored tokens cannot be taken back, got {n}")
        self._check()
        self.cache._reserve(self.ids, n)
        self.cache._advance(self.ids, n)

    def begin(self, n: int) -> "PagedStep":
        """Reserves pages for ``n`` tokens per sequence and lays out where they go."""
        c, ids = self.cache, self.ids
        if n < 1 or not len(ids):
            raise ValueError(f"a forward needs sequences and tokens, got {len(ids)} of {n} tokens")
        self._check()
        c._reserve(ids, n)
        B, ps = len(ids), c.page_size
        pos = c._len[ids][:, None] + np.arange(n)[None]
        slots = c._table[ids[:, None], pos // ps].astype(np.int64) * ps + pos % ps
        cols = int(pos[:, -1].max()) // ps + 1
        where = np.stack((pos.reshape(-1), slots.reshape(-1)))
        meta = np.concatenate((pos[:, -1] + 1, np.arange(B + 1) * n, c._table[ids, :cols].reshape(-1))).astype(np.int32)
        where, meta = (torch.from_numpy(x).to(c.device) for x in (where, meta))
        return PagedStep(c, n, where[0], where[1], meta[:B], meta[B:2 * B + 1], meta[2 * B + 1:].view(B, cols),
                         int(pos[:, -1].max()) + 1)


class PagedStep:
    """Where one forward's tokens go, on the device; the layers' ``k_cache``."""

    def __init__(self, cache, n, positions, slots, kv_lens, q_offsets, page_table, max_len):
        self.cache, self.n, self.positions, self.slots = cache, n, positions, slots
        self.kv_lens, self.q_offsets, self.page_table, self.max_len = kv_lens, q_offsets, page_table, max_len

    def layer(self, l: int) -> "PagedLayer":
        return PagedLayer(self, self.cache.k_pages[l], self.cache.v_pages[l])


class PagedLayer:
    def __init__(self, step: PagedStep, k_pages, v_pages):
        self.step, self.k_pages, self.v_pages = step, k_pages, v_pages
        self.dtype = k_pages.dtype

    def attend(self, q, k, v):
        """Stores k, v and attends: q, k, v [N, H, hd] (rotated; any strides) -> [N, H, hd]."""
        s, c = self.step, self.step.cache
        ops.paged_append(None, k, v, self.k_pages, self.v_pages, s.slots, err=c.err)
        kw = dict(window=c.window, sinks=c.sinks, err=c.err)
        if s.n == 1:
            return ops.paged_attention(q, self.k_pages, self.v_pages, s.page_table, s.kv_lens, max_len=s.max_len, **kw)
        # prompts as over the dense cache, whose kernels round the probabilities once too
        return ops.paged_prefill_attention(q, s.q_offsets, self.k_pages, self.v_pages, s.page_table, s.kv_lens,
                                           max_q=s.n, rounded=True, **kw)
