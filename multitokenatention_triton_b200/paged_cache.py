"""A paged cache for token-by-token generation: which pages belong to which sequence, and the device tensors that the kernels read.

The reference has no cache: it generates by running the whole prefix again.  Here a sequence keeps its keys and values in pages of
`page_size` tokens, and the last `history` queries, which the convs of the following tokens look back on (`query_history` of the
attention modules).  Sequences that were forked share pages until one of them writes into a shared one.

Page numbers, lengths and reference counts live on the host, where pages are handed out; tables and lengths are mirrored into device
tensors that stay where they are, so that a captured graph of a decoding step follows them.  All device work is enqueued on the
current stream of the cache's device: calls from several streams are ordered by the caller.
"""
from __future__ import annotations

import heapq
import itertools
import operator
from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Set, Tuple, Union

import torch

from . import ops
from ._lib import MTALibraryError, cache_status


_STAMPS = itertools.count(1)             # of all caches, so that a batch is known by its own cache only


class CacheFullError(MTALibraryError):
    """No page or no slot is left for what was asked; the cache is as it was."""


@dataclass(frozen=True)
class CacheBatch:
    """New tokens of some sequences, as PagedKVCache.extend() reserved them: batch row b is sequence slots[b], which has lengths[b] tokens, the last
    counts[b] of them new.  slot_ids and count_ids are the same on the device."""
    slots: Tuple[int, ...]
    counts: Tuple[int, ...]
    lengths: Tuple[int, ...]
    max_length: int
    slot_ids: torch.Tensor
    count_ids: torch.Tensor
    stamps: Tuple[int, ...]

    @property
    def from_empty(self) -> bool:
        """Whether every sequence had no token before."""
        return self.counts == self.lengths

    def without_padding(self, *tokens: torch.Tensor) -> Tuple[torch.Tensor, ...]:
        """(B,heads,T,D) tensors with zeros behind every row's count, the same ones where there is nothing behind.  The whole-sequence forwards
        multiply what lies behind a row with zeros, which leaves NaN of what is not finite, and padding may be anything."""
        T = tokens[0].shape[2]
        if min(self.counts, default=T) >= T:
            return tokens
        behind = torch.arange(T, device=self.count_ids.device) >= self.count_ids[:, None]
        return tuple(t.masked_fill(behind[:, None, :, None], 0.0) for t in tokens)


def expand_heads(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Keys and values of shared heads repeated for every query head, as the whole-sequence forwards take them."""
    group = q.shape[1] // k.shape[1]
    return (q, k, v) if group <= 1 else (q, k.repeat_interleave(group, dim=1), v.repeat_interleave(group, dim=1))


class PagedKVCache:
    """n_layers caches with one table: k_pages, v_pages (layers, pages, kv heads, page, D), q_hist (layers, sequences, history, H, D),
    table (sequences, pages of the longest), lengths (sequences).  Tokens reach them through append(); a program that writes them itself (a saved
    prefix, say) takes them from layer(), which says so."""

    def __init__(self, n_heads: int, head_dim: int, num_pages: int, max_sequences: int, max_length: int, history: int, page_size: int = 64,
                 n_kv_heads: Optional[int] = None, n_layers: int = 1, dtype: torch.dtype = torch.bfloat16, device: Union[str, torch.device] = "cuda"):
        kv = n_heads if n_kv_heads is None else n_kv_heads
        if min(n_heads, head_dim, num_pages, max_sequences, max_length, history, kv, n_layers) < 1:
            raise MTALibraryError("PagedKVCache: all sizes are positive")
        if n_heads % kv:
            raise MTALibraryError(f"PagedKVCache: {n_heads} heads are no multiple of {kv} key-value heads")
        if not 16 <= page_size <= 65536 or page_size & (page_size - 1):
            raise MTALibraryError(f"PagedKVCache: a page of {page_size} tokens; a power of two from 16 to 65536 is wanted")
        if dtype not in ops._lib.DTYPE_CODE or head_dim % 8 or head_dim > (128 if dtype == torch.float32 else 256):
            raise MTALibraryError(f"PagedKVCache: head dimension {head_dim} in {dtype}; a multiple of 8 up to 256 (float32: 128) in float32, bfloat16 or "
                                  "float16 is wanted")
        self.n_heads, self.n_kv_heads, self.head_dim, self.page_size, self.history = n_heads, kv, head_dim, page_size, history
        self.num_pages, self.max_sequences, self.n_layers = num_pages, max_sequences, n_layers
        width = -(-max_length // page_size)
        if width * page_size > 1 << 30 or n_layers > 16384:
            raise MTALibraryError(f"PagedKVCache: {n_layers} layers of sequences of {max_length} tokens; up to 16384 layers and 2^30 tokens are supported")
        row = head_dim * dtype.itemsize
        if kv * page_size * row > 1 << 30 or history * n_heads * row > 1 << 30:
            raise MTALibraryError(f"PagedKVCache: a page of {kv * page_size * row} bytes and {history * n_heads * row} bytes of queries a sequence; up to 1 GiB is "
                                  "supported")
        self.max_length = max_length
        with torch.device(device):
            self.k_pages = torch.empty(n_layers, num_pages, kv, page_size, head_dim, dtype=dtype)
            self.v_pages = torch.empty_like(self.k_pages)
            self.q_hist = torch.empty(n_layers, max_sequences, history, n_heads, head_dim, dtype=dtype)
            self.table = torch.zeros(max_sequences, width, dtype=torch.int32)
            self.lengths = torch.zeros(max_sequences, dtype=torch.int32)
        self.device = self.k_pages.device
        self._free_pages: List[int] = list(range(num_pages))              # a heap: the lowest page is handed out first
        self._free_slots: List[int] = list(range(max_sequences))
        self._refs = [0] * num_pages
        self._pages: List[Optional[List[int]]] = [None] * max_sequences   # of each sequence, in order; None: the slot is free
        self._len = [0] * max_sequences
        self._stamp = dict.fromkeys(range(max_sequences), 0)              # of each slot; a new one whenever a sequence's tokens or pages change
        self._captured: List[CacheBatch] = []                             # whose ids graphs read
        # What append() has written: per layer the tokens of each slot.  Not judged by it: slots that replays of a graph write (`_replayed`) and
        # layers whose tensors were handed out (not `_seen`).  `_high`: how far a sequence's queries went before it was truncated.
        self._written: List[Dict[int, int]] = [dict.fromkeys(range(max_sequences), 0) for _ in range(n_layers)]
        self._seen = [True] * n_layers
        self._high = [0] * max_sequences
        self._replayed: Set[int] = set()                                  # slots that a captured append names

    # ---- what is there -------------------------------------------------------------------------------------------------

    def length(self, slot: int) -> int:
        self._check(slot)
        return self._len[slot]

    @property
    def free_pages(self) -> int:
        return len(self._free_pages)

    @property
    def free_slots(self) -> int:
        return len(self._free_slots)

    def _check(self, slot: int) -> None:
        if not 0 <= slot < self.max_sequences or self._pages[slot] is None:
            raise MTALibraryError(f"slot {slot} holds no sequence")

    # ---- sequences -----------------------------------------------------------------------------------------------------

    def add(self) -> int:
        """A new sequence of no tokens; returns its slot."""
        if not self._free_slots:
            raise CacheFullError(f"all {self.max_sequences} sequences of the cache are in use")
        slot = heapq.heappop(self._free_slots)
        self._pages[slot] = []
        self._len[slot] = 0
        for written in self._written:
            written[slot] = 0
        self._high[slot] = 0
        self._stamp[slot] = next(_STAMPS)
        return slot

    def free(self, slot: int) -> None:
        """Ends a sequence.  Its pages are free once no fork of it holds them."""
        self._check(slot)
        for p in self._pages[slot]:
            self._release(p)
        self._pages[slot] = None
        self._stamp[slot] = next(_STAMPS)
        heapq.heappush(self._free_slots, slot)
        self._upload([(slot, 0)], [])

    def _release(self, page: int) -> None:
        self._refs[page] -= 1
        if self._refs[page] == 0:
            heapq.heappush(self._free_pages, page)

    def extend(self, slots: Sequence[int], counts: Union[int, Sequence[int]]) -> CacheBatch:
        """Makes room for counts[b] new tokens of sequence slots[b] (one number: the same for all) and returns the batch to append and attend with.
        A page that a fork shares is copied before it is written.  Raises CacheFullError, with nothing changed, when pages or the
        longest length do not suffice.  The tokens count from now on: truncate() takes back those that are not appended after all."""
        slots = tuple(int(s) for s in slots)
        counts = (int(counts),) * len(slots) if isinstance(counts, int) else tuple(int(n) for n in counts)
        if len(counts) != len(slots) or any(n < 1 for n in counts):
            raise MTALibraryError(f"extend: {len(slots)} sequences need one positive count each, got {counts}")
        if len(set(slots)) < len(slots):
            raise MTALibraryError("extend: a sequence stands in the batch twice")
        need = 0
        refs = {}                                          # what is left of the counts of shared pages when they are copied one by one
        own: List[bool] = []
        for s, n in zip(slots, counts):
            self._check(s)
            total = self._len[s] + n
            if total > self.max_length:
                raise CacheFullError(f"extend: sequence {s} would have {total} tokens, the cache's longest are {self.max_length}")
            need += -(-total // self.page_size) - len(self._pages[s])
            own.append(False)
            if self._len[s] % self.page_size:
                last = self._pages[s][-1]
                left = refs.get(last, self._refs[last])
                if left > 1:                               # the last holder that writes keeps the page itself
                    own[-1] = True
                    refs[last] = left - 1
                    need += 1
        if need > len(self._free_pages):
            raise CacheFullError(f"extend: {need} pages are needed, {len(self._free_pages)} are free")
        copies, entries, lengths = [], [], []
        for s, n, copy in zip(slots, counts, own):
            pages = self._pages[s]
            if copy:
                fresh = heapq.heappop(self._free_pages)
                self._refs[fresh] = 1
                copies.append((pages[-1], fresh))
                self._release(pages[-1])
                pages[-1] = fresh
                entries.append((s, len(pages) - 1, fresh))
            self._len[s] += n
            while len(pages) * self.page_size < self._len[s]:
                fresh = heapq.heappop(self._free_pages)
                self._refs[fresh] = 1
                entries.append((s, len(pages), fresh))
                pages.append(fresh)
            self._stamp[s] = next(_STAMPS)
            lengths.append(self._len[s])
        if copies:
            self._copy(copies, [])
        self._upload(list(zip(slots, lengths)), entries)
        ids = self._ints(slots + counts)
        return CacheBatch(slots, counts, tuple(lengths), max(lengths, default=0), ids[:len(slots)], ids[len(slots):], tuple(self._stamp[s] for s in slots))

    def fork(self, slot: int, n: int = 1) -> List[int]:
        """n copies of a sequence, which share its pages; returns their slots.  Only its queries are copied now, so a batch of the sequence that
        extend() gave before is stale: what is appended later would reach the shared pages, but not the copies' queries."""
        self._check(slot)
        if n < 0:
            raise MTALibraryError(f"fork: {n} copies")
        if n > len(self._free_slots):
            raise CacheFullError(f"fork: {n} sequences are wanted, {len(self._free_slots)} slots are free")
        made = []
        for _ in range(n):
            new = heapq.heappop(self._free_slots)
            self._pages[new] = list(self._pages[slot])
            for p in self._pages[new]:
                self._refs[p] += 1
            self._len[new] = self._len[slot]
            for written in self._written:
                written[new] = self._len[slot] if slot in self._replayed else written[slot]
            self._high[new] = self._high[slot]
            self._stamp[new] = next(_STAMPS)
            made.append(new)
        if made:
            self._stamp[slot] = next(_STAMPS)
            self._upload([(s, self._len[s]) for s in made], [(s, i, p) for s in made for i, p in enumerate(self._pages[s])])
            if self._len[slot]:
                self._copy([], [(slot, s) for s in made])
        return made

    def truncate(self, slot: int, length: int) -> None:
        """Takes back what a sequence has behind its first `length` tokens, so that others can follow them: tokens that extend() reserved and whose
        append was refused or never came, the newest token, or all.  The cache keeps the last `history` queries, and writing a token drops
        the oldest: further back than one written token it goes only to 0 or while no query has been dropped yet."""
        self._check(slot)
        if not 0 <= length <= self._len[slot]:
            raise MTALibraryError(f"truncate: sequence {slot} has {self._len[slot]} tokens, {length} were to be left")
        if length == self._len[slot]:
            return
        # of what was not seen whatever was reserved may have been written
        high = max(self._high[slot], max(written[slot] if seen and slot not in self._replayed else self._len[slot]
                                         for written, seen in zip(self._written, self._seen)))
        if length and high > self.history and length < high - 1:
            raise MTALibraryError(f"truncate: the queries before token {length} of sequence {slot} are gone: {high} tokens were written, the cache keeps the last "
                                  f"{self.history}")
        pages, keep = self._pages[slot], -(-length // self.page_size)
        for p in pages[keep:]:
            self._release(p)
        del pages[keep:]
        self._len[slot] = length
        self._high[slot] = high if length else 0
        for written in self._written:
            written[slot] = min(written[slot], length)
        self._stamp[slot] = next(_STAMPS)
        self._upload([(slot, length)], [])

    def compact(self) -> int:
        """Moves the pages in use to the front of the pools; returns how many there are.  Batches that extend() gave before are stale."""
        used = self.num_pages - len(self._free_pages)
        moves = dict(self._moves())
        if moves:
            self._copy(list(moves.items()), [])
            entries = []
            for s, pages in enumerate(self._pages):
                if pages is None or not any(p in moves for p in pages):
                    continue
                entries += [(s, i, moves[p]) for i, p in enumerate(pages) if p in moves]
                self._pages[s] = [moves.get(p, p) for p in pages]
                self._stamp[s] = next(_STAMPS)
            for a, b in moves.items():
                self._refs[b], self._refs[a] = self._refs[a], 0
            self._free_pages = list(range(used, self.num_pages))
            self._upload([], entries)
        return used

    def _moves(self) -> List[Tuple[int, int]]:
        """(page behind the front part, free page in it) pairs: no page is both, so that they can be copied at once."""
        used = self.num_pages - len(self._free_pages)
        holes = sorted(p for p in self._free_pages if p < used)
        return list(zip((p for p in range(used, self.num_pages) if self._refs[p]), holes))

    # ---- device work ---------------------------------------------------------------------------------------------------

    def _ints(self, values: Sequence[int], dtype: torch.dtype = torch.int32) -> torch.Tensor:
        t = torch.tensor(list(values), dtype=dtype)
        if self.device.type != "cuda":
            return t
        # page-locked, so that the copy waits for nothing; torch keeps the memory until the copy has run
        return t.pin_memory().to(self.device, non_blocking=True) if t.numel() else t.to(self.device)

    def _upload(self, lengths: Sequence[Tuple[int, int]], entries: Sequence[Tuple[int, int, int]]) -> None:
        """(slot, tokens) pairs and (slot, index, page) triples into the device's lengths and table."""
        if not lengths and not entries:
            return
        width = self.table.shape[1]
        at = self._ints([s for s, _ in lengths] + [s * width + i for s, i, _ in entries] + [n for _, n in lengths] + [p for _, _, p in entries], torch.int64)
        a, b = len(lengths), len(entries)
        if a:
            self.lengths.index_copy_(0, at[:a], at[a + b:a + b + a].int())
        if b:
            self.table.view(-1).index_copy_(0, at[a:a + b], at[a + b + a:].int())

    def _copy(self, pages: Sequence[Tuple[int, int]], slots: Sequence[Tuple[int, int]]) -> None:
        ids = self._ints([a for a, _ in pages] + [b for _, b in pages] + [a for a, _ in slots] + [b for _, b in slots])
        n, m = len(pages), len(slots)
        ops.cache_copy(self.k_pages, self.v_pages, ids[:n], ids[n:2 * n], self.q_hist, ids[2 * n:2 * n + m], ids[2 * n + m:])

    def layer(self, layer: int) -> Tuple[torch.Tensor, ...]:
        """(q_hist, k_pages, v_pages, table, lengths) of one layer, as ops.cache_append and the decoding calls take them.  Whoever takes them may
        write them: append() no longer asks whether all earlier tokens of this layer went through it."""
        tensors = self._layer(layer)
        self._seen[layer] = False
        return tensors

    def _check_layer(self, layer: int) -> None:
        if not 0 <= layer < self.n_layers:
            raise MTALibraryError(f"layer {layer} of a cache of {self.n_layers}")

    def _layer(self, layer: int) -> Tuple[torch.Tensor, ...]:
        self._check_layer(layer)
        return self.q_hist[layer], self.k_pages[layer], self.v_pages[layer], self.table, self.lengths

    def check_batch(self, batch: CacheBatch) -> None:
        """Raises if a sequence of the batch was extended, forked, truncated, freed or moved after extend() gave it, or if another cache's did."""
        if tuple(map(self._stamp.get, batch.slots)) != batch.stamps:
            changed = [s for s, stamp in zip(batch.slots, batch.stamps) if self._stamp.get(s) != stamp]
            raise MTALibraryError(f"the batch is stale: sequence {changed[0]} has changed since extend(), or is another cache's")

    def longest(self, batch: CacheBatch, max_length: Optional[int]) -> int:
        """The longest length that an attention call over the batch is to serve: the batch's own, or a larger one."""
        if max_length is None:
            return batch.max_length
        if not batch.max_length <= max_length <= self.max_length:
            raise MTALibraryError(f"max_length = {max_length}, but the batch has {batch.max_length} tokens and the cache at most {self.max_length}")
        return max_length

    def check_reader(self, what: str, n_heads: int, history: int) -> None:
        """Raises if an attention module of n_heads heads that looks back on `history` queries cannot read this cache."""
        if n_heads != self.n_heads or history > self.history:
            raise MTALibraryError(f"{what}: {n_heads} heads that look back on {history} queries, but the cache has {self.n_heads} heads and keeps {self.history} queries")

    def check_step(self, batch: CacheBatch, xk: torch.Tensor, layer: int = 0) -> None:
        """Raises where append() would: the batch is stale, the tokens are not the batch's, or tokens before them were never written."""
        self.check_batch(batch)
        if xk.dim() != 4 or xk.shape[0] != len(batch.slots) or (batch.counts and max(batch.counts) > xk.shape[2]):
            raise MTALibraryError(f"append: keys {tuple(xk.shape)} for {len(batch.slots)} sequences with up to {max(batch.counts, default=0)} new tokens")
        self._check_layer(layer)
        if self._seen[layer]:
            written = self._written[layer]
            if not any(map(operator.lt, map(written.get, batch.slots), map(operator.sub, batch.lengths, batch.counts))):
                return
            for s, n, total in zip(batch.slots, batch.counts, batch.lengths):
                if written[s] < total - n and s not in self._replayed:
                    raise MTALibraryError(f"append: of the {total - n} tokens that sequence {s} had before, layer {layer} was given {written[s]}: append "
                                          "what extend() reserved, or take it back with truncate()")

    def append(self, batch: CacheBatch, xk: torch.Tensor, xv: torch.Tensor, xq: torch.Tensor, layer: int = 0) -> None:
        """Writes the batch's new tokens of one layer: xk, xv (B,kv heads,T,D), xq (B,H,T,D) with T >= every count; tokens behind a row's count are
        not read.  Raises if tokens before them were reserved and never written, which the attention would read.  Inside a graph capture the
        cache keeps the batch's ids for as long as it lives itself: replays write the newest tokens of the same sequences."""
        self._append(batch, xk, xv, xq, layer, self._layer(layer))

    def _append(self, batch: CacheBatch, xk: torch.Tensor, xv: torch.Tensor, xq: torch.Tensor, layer: int, tensors: Tuple[torch.Tensor, ...]) -> None:
        self.check_step(batch, xk, layer)
        q_hist, k_pages, v_pages, table, lengths = tensors
        capturing = self._capturing()
        if capturing and (not self._captured or self._captured[-1] is not batch):
            self._captured.append(batch)                    # the graph's replays read its ids, which the caller need not keep
        ops.cache_append(xk, xv, xq, k_pages, v_pages, q_hist, table, lengths, slots=batch.slot_ids, counts=batch.count_ids)
        self._written[layer].update(zip(batch.slots, batch.lengths))
        if capturing:
            self._replayed.update(batch.slots)

    def _capturing(self) -> bool:
        return self.device.type == "cuda" and torch.cuda.is_current_stream_capturing()

    def check(self) -> None:
        """Waits for the device and raises if a call over the cache met something out of range (a table or lengths written by other hands)."""
        cache_status(self.device)
