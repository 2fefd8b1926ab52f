"""A paged key-value cache for a batch of sequences and all layers of a model.

:class:`~dcr_b200.kv_cache.StaticKVCache` gives every sequence of a layer ``N_max`` positions from
the start; :class:`PagedKVCache` hands out pages of ``page_size`` slots as sequences grow, takes
them back when a sequence ends or its slots are evicted, and keeps one page table for all layers
(a page number means the same page of every layer's pool). With a ``budget`` it also keeps, per
layer, the accumulated attention weight and the position of every slot, and evicts what is over
the budget (``paged_evict``). Without one, sequences may share the pages of a common prefix
(:meth:`PagedKVCache.fork`), which attention then reads once for them where that pays
(``paged_shared_attention``). The reference concatenates one contiguous cache per layer
(dcr_attention/models/llama/compat.py:208-254) and has no counterpart.

The host knows every length, so page handling never waits for the device; lengths, slots and
positions are also on the device, where the kernels read them.
"""
from __future__ import annotations

from itertools import accumulate
from typing import List, Optional, Sequence

import torch

from dcr_b200.kernel.cuda._common import HEAD_DIM, check_dtype, require
from dcr_b200.kernel.cuda.paged import (PAGED_HEAD_DIMS, paged_append, paged_attention,
                                        paged_evict, paged_prefill, paged_rotary_append,
                                        paged_shared_attention)


# Bytes of keys and values that the shared call has to save a layer for :meth:`PagedKVCache.attend` to take
# it instead of the plain one, by the bytes of an element. It has a fixed cost of its own (the prefix's
# kernel, parts and a join beside the own slots' kernels). Measured on cold pools, plain -> shared: in 16 bits
# 51 MB 18 -> 31 us, 101 MB 27 -> 36, 126 MB 29 -> 24 to 36 -> 49, 201 MB 41 -> 40, 252 MB 47 -> 30 to 53 ->
# 53, 528 MB 90 -> 43, 2.1 GB 310 -> 57 (32 query heads of 64 or 64 of 128, on 4 and 8, 2 to 64 sequences); in 32 bits,
# bound by arithmetic, 503 MB 121 -> 198, 1.0 GB 137 -> 162 to 230 -> 141, 2.1 GB 275 -> 172.
SHARED_BYTES = {2: 200e6, 4: 1e9}


class PagedKVCache:
    """Pools of ``pages`` pages for ``layers`` layers and up to ``batch`` sequences of at most
    ``max_slots`` cached slots each.

    ``budget``: most slots a sequence keeps per layer and KV head after an eviction, of which
    the first ``sinks`` positions and the ``recent`` last ones are never evicted; an eviction runs
    when a sequence holds ``budget + slack`` slots or more."""

    def __init__(self, layers: int, batch: int, H_kv: int, pages: int, max_slots: int, *,
                 page_size: int = 64, D: int = HEAD_DIM, dtype: torch.dtype, device,
                 budget: Optional[int] = None, sinks: int = 4, recent: int = 64, slack: int = 1):
        self.device = torch.device(device)
        check_dtype(torch.empty(0, dtype=dtype), "cache")
        require(D in PAGED_HEAD_DIMS, f"head dim must be one of {PAGED_HEAD_DIMS}, got {D}")
        require(layers > 0 and batch > 0 and H_kv > 0 and pages > 0 and page_size > 0 and
                max_slots > 0, "layers, batch, H_kv, pages, page_size and max_slots must be positive")
        if budget is not None:
            require(0 < budget < max_slots, f"budget must be in (0, max_slots={max_slots})")
            require(slack > 0 and budget + slack <= max_slots, "budget + slack must fit max_slots")
            require(0 <= sinks and 0 <= recent and sinks + recent <= budget,
                    "sinks + recent must fit the budget")
        self.batch, self.H_kv, self.D, self.page_size, self.dtype = batch, H_kv, D, page_size, dtype
        self.max_pages = -(-max_slots // page_size)
        self.max_slots, self.budget, self.sinks, self.recent, self.slack = (max_slots, budget, sinks,
                                                                            recent, slack)
        shape = (pages, H_kv, page_size, D)
        self.k = [torch.empty(shape, dtype=dtype, device=self.device) for _ in range(layers)]
        self.v = [torch.empty(shape, dtype=dtype, device=self.device) for _ in range(layers)]
        i32 = dict(dtype=torch.int32, device=self.device)
        self.page_table = torch.full((batch, self.max_pages), -1, **i32)
        self.lengths = torch.zeros(batch, **i32)     # cached slots
        self.seen = torch.zeros(batch, **i32)        # positions so far
        self.queried = torch.zeros(batch, **i32)     # lengths of the sequences that grew last, else 0
        self.starts = torch.zeros(batch + 1, **i32)  # where each one's tokens reserved last begin
        self._begins = [0] * (batch + 1)             # starts, as published
        self.groups = self.prefix = None             # sequences that share pages (fork), of the next two
        self._groups, self._prefix = torch.zeros(batch + 1, **i32), torch.zeros(batch, **i32)
        self._spans = torch.zeros(batch + 1, **i32)  # groups without those that share nothing
        self._host_spans, self._host_prefix = [0, batch], [0] * batch
        self._saved = {}                             # by window: bytes that sharing saves a call, as it stands
        self.shared_bytes = SHARED_BYTES[dtype.itemsize]
        self.weights = self.pos = None
        if budget is not None:
            tables = (batch, H_kv, self.max_pages * page_size)
            f32 = dict(dtype=torch.float32, device=self.device)
            self.weights = [torch.zeros(tables, **f32) for _ in range(layers)]
            self.pos = [torch.zeros(tables, **i32) for _ in range(layers)]
            self._provisional = {}  # sequence: its layers' weights before a prompt's last token counted
            self._spare_weights, self._spare_pos = torch.zeros(tables, **f32), torch.zeros(tables, **i32)
        self.free_pages = list(range(pages - 1, -1, -1))
        self.host_lengths = [0] * batch
        self.host_seen = [0] * batch
        self._grew = [False] * batch                 # the sequences that reserved a token last
        self.host_pages: List[List[int]] = [[] for _ in range(batch)]
        self._mapped = [0] * batch                   # pages of each one in the page table
        self._intact = [0] * batch                   # the first of these that it still holds
        self._holders = [0] * pages                  # sequences that hold each page
        self._shared = 0                             # pages that several hold
        self._tokens = None  # (seq, slots, positions) of the tokens reserved last

    # ------------------------------------------------------------------------------- host side
    def _to_device(self, dst: torch.Tensor, values: Sequence[int]) -> None:
        """Copies values into dst in the current stream's order, without waiting for it."""
        src = torch.tensor(values, dtype=torch.int32)
        pinned = self.device.type == "cuda"
        dst.copy_(src.pin_memory() if pinned else src, non_blocking=pinned)

    def _publish(self, rows: Sequence[int]) -> None:
        """Copies the host's lengths and what changed in the page table's given rows to the device."""
        self._saved = {}
        self._to_device(self.lengths, self.host_lengths)
        self._to_device(self.seen, self.host_seen)
        self._to_device(self.queried, [n if g else 0 for n, g in zip(self.host_lengths, self._grew)])
        for b in rows:
            held, first = self.host_pages[b], self._intact[b]
            last = max(len(held), self._mapped[b])
            if first < last:
                self._to_device(self.page_table[b, first:last], held[first:] + [-1] * (last - len(held)))
            self._mapped[b] = self._intact[b] = len(held)

    def _regroup(self) -> None:
        """Publishes the groups that share pages. What sequences share changes when one is forked or
        released: a page that one grows into is its own, so its prefix stays what it is."""
        groups, prefix = self.shared_groups()
        self._saved = {}
        if not any(prefix):  # nobody shares, or no neighbours do
            self.groups = self.prefix = None
            return
        self._to_device(self._prefix, prefix)
        self.groups, self.prefix = self._groups[:len(groups)], self._prefix
        self._to_device(self.groups, groups)
        # What attend passes: a group that shares nothing joins the one before it, or those before the first
        # that shares are one, since a call of many groups does not cut their prefixes up.
        self._host_spans = [0, *(b for b in groups[1:-1] if prefix[b]), self.batch]
        self._host_prefix = prefix
        self._to_device(self._spans[:len(self._host_spans)], self._host_spans)

    def _shares(self, b: int) -> bool:
        """Whether another sequence holds sequence b's first page."""
        held = self.host_pages[b]
        return bool(held) and self._holders[held[0]] > 1

    def _common(self, a: int, b: int) -> int:
        """First pages that sequences a and b both hold, by bisection: with one they hold all before it."""
        x, y = self.host_pages[a], self.host_pages[b]
        least, most = 0, min(len(x), len(y))
        while least < most:
            mid = (least + most + 1) // 2
            if x[mid - 1] == y[mid - 1]:
                least = mid
            else:
                most = mid - 1
        return least

    def shared_groups(self):
        """(groups, prefix), as :func:`paged_shared_attention` takes them: neighbouring sequences whose
        first pages are the same ones, and the slots in them. A sequence that shares nothing, since it has
        ended, waits or grew from a prompt of its own, does not part its neighbours: it stays in their
        group with a prefix of 0. The pages are the group's first sequence's, so those before the first
        that shares are alone."""
        groups, prefix, lead = [0], [0] * self.batch, None
        for b in range(self.batch):
            same = 0
            if self._shares(b):
                same = 0 if lead is None else self._common(lead, b)
                if same == 0:
                    lead = b
            elif lead is not None:
                continue
            if same == 0:
                if b > 0:
                    groups.append(b)
            else:
                prefix[b] = same * self.page_size
                prefix[lead] = max(prefix[lead], prefix[b])
        return groups + [self.batch], prefix

    def _shared_call_pays(self, window: int) -> bool:
        """Whether reading the shared pages once for the sequences that grew last saves so much."""
        if window not in self._saved:
            n, slots = [x if g else 0 for x, g in zip(self.host_lengths, self._grew)], 0
            for a, b in zip(self._host_spans, self._host_spans[1:]):
                seen = [max(0, min(self._host_prefix[s], n[s]) - (max(0, n[s] - window) if window else 0))
                        for s in range(a, b)]
                slots += sum(seen) - max(seen)
            self._saved[window] = slots * 2 * self.H_kv * self.D * self.dtype.itemsize
        return self._saved[window] >= self.shared_bytes

    def _resize(self, b: int, length: int) -> bool:
        """Gives sequence b the pages of `length` slots; True if they changed."""
        need, held = -(-length // self.page_size), self.host_pages[b]
        before = len(held)
        while len(held) < need:
            held.append(self.free_pages.pop())
            self._holders[held[-1]] = 1
        while len(held) > need:
            page = held.pop()
            self._holders[page] -= 1
            if self._holders[page] == 0:
                self.free_pages.append(page)
            elif self._holders[page] == 1:
                self._shared -= 1
        self._intact[b] = min(self._intact[b], len(held))
        self.host_lengths[b] = length
        return len(held) != before

    def reserve(self, new_tokens: Sequence[int]) -> int:
        """Makes room for ``new_tokens[b]`` more tokens of every sequence b: pages, lengths and the
        (sequence, slot, position) of each token in sequence order, which :meth:`append` uses for
        every layer. Returns the number of tokens. Refuses, changing nothing, where a sequence
        would pass ``max_slots`` or the pool runs out of pages."""
        require(len(new_tokens) == self.batch and all(n >= 0 for n in new_tokens),
                f"new_tokens must be {self.batch} counts")
        want = [self.host_lengths[b] + n for b, n in enumerate(new_tokens)]
        require(max(want) <= self.max_slots,
                f"sequence {want.index(max(want))} would hold {max(want)} of {self.max_slots} slots")
        pages = sum(-(-n // self.page_size) - len(self.host_pages[b]) for b, n in enumerate(want))
        require(pages <= len(self.free_pages),
                f"{pages} pages needed, {len(self.free_pages)} free")
        seq = [b for b, n in enumerate(new_tokens) for _ in range(n)]
        slots = [self.host_lengths[b] + i for b, n in enumerate(new_tokens) for i in range(n)]
        positions = [self.host_seen[b] + i for b, n in enumerate(new_tokens) for i in range(n)]
        changed = [b for b, n in enumerate(want) if self._resize(b, n)]
        self.host_seen = [s + n for s, n in zip(self.host_seen, new_tokens)]
        self._grew = [n > 0 for n in new_tokens]
        self._publish(changed)
        i32 = dict(dtype=torch.int32)
        begins = [0, *accumulate(new_tokens)]
        if begins != self._begins:  # the same from one decode step to the next
            self._to_device(self.starts, begins)
            self._begins = begins
        self._tokens = tuple(torch.tensor(x, **i32).to(self.device) for x in (seq, slots, positions))
        return len(seq)

    def release(self, b: int) -> None:
        """Ends sequence b: its pages go back to the pool."""
        shared = self._shared
        self._resize(b, 0)
        if self.budget is not None:
            self._provisional.pop(b, None)
        self.host_seen[b], self._grew[b] = 0, False
        self._publish([b])
        if shared:
            self._regroup()

    def fork(self, b: int, others: Sequence[int]) -> None:
        """Gives the empty sequences ``others`` what sequence b holds: its full pages are shared, the
        last one, if it is not full, is copied. A page goes back to the pool with the last sequence
        that holds it. What was reserved last has to be appended in every layer before. Refuses, changing
        nothing, where the pool runs out of pages."""
        require(self.budget is None, "a cache with a budget shares no pages")
        require(0 <= b < self.batch and self.host_lengths[b] > 0, f"sequence {b} holds nothing")
        require(len(set(others)) == len(others) and
                all(0 <= o < self.batch and o != b and self.host_lengths[o] == 0 for o in others),
                "others must be different empty sequences")
        n, pages = self.host_lengths[b], self.host_pages[b]
        full = n // self.page_size
        copies = len(others) if n % self.page_size else 0
        require(copies <= len(self.free_pages), f"{copies} pages needed, {len(self.free_pages)} free")
        for o in others:
            self.host_pages[o] = pages[:full]
            for page in pages[:full]:
                self._holders[page] += 1
                self._shared += self._holders[page] == 2
            self._resize(o, n)
            self.host_seen[o] = self.host_seen[b]
            self._grew[o] = False
        if copies:
            to = torch.tensor([self.host_pages[o][-1] for o in others], device=self.device)
            for pool in self.k + self.v:
                pool[to] = pool[pages[full]].clone()
        self._publish(others)
        self._regroup()

    def over_budget(self) -> bool:
        """Whether some sequence holds ``budget + slack`` slots or more."""
        return self.budget is not None and max(self.host_lengths) >= self.budget + self.slack

    # ----------------------------------------------------------------------------- device side
    def append(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               cos: torch.Tensor, sin: torch.Tensor, *, q_weight: Optional[torch.Tensor] = None,
               k_weight: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
        """The layer's queries, keys and values of the tokens reserved last: norms (with weights),
        rotation by the tokens' positions, append; returns the rotated queries."""
        require(self._tokens is not None, "reserve() comes before append()")
        seq, slots, positions = self._tokens
        return paged_append(q, k, v, cos, sin, positions, self.k[layer], self.v[layer],
                            self.page_table, slots, seq=seq, q_weight=q_weight, k_weight=k_weight,
                            eps=eps, weights=None if self.weights is None else self.weights[layer],
                            pos=None if self.pos is None else self.pos[layer])

    def append_rotary(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                      inv_freq: torch.Tensor, *, interleaved: bool = False, factor: float = 1.0,
                      q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                      eps: float = 1e-5) -> torch.Tensor:
        """:meth:`append` with the rotation of :func:`paged_rotary_append`: from frequencies, in any
        layout."""
        require(self._tokens is not None, "reserve() comes before append_rotary()")
        seq, slots, positions = self._tokens
        return paged_rotary_append(q, k, v, inv_freq, positions, self.k[layer], self.v[layer],
                                   self.page_table, slots, seq=seq, interleaved=interleaved, factor=factor,
                                   q_weight=q_weight, k_weight=k_weight, eps=eps,
                                   weights=None if self.weights is None else self.weights[layer],
                                   pos=None if self.pos is None else self.pos[layer])

    def prefill_attend(self, layer: int, q: torch.Tensor, *, window: int = 0) -> torch.Tensor:
        """O ``[tokens, H, D]`` of the tokens reserved last, each over its sequence's slots up to its own.
        No attention weights are accumulated (:meth:`weigh`)."""
        require(self._tokens is not None, "reserve() comes before prefill_attend()")
        return paged_prefill(q, self.k[layer], self.v[layer], self.page_table, self.lengths, self.starts,
                             window=window)

    def attend(self, layer: int, q: torch.Tensor, *, window: int = 0) -> torch.Tensor:
        """O ``[batch, H, D]`` of one query row per sequence over the layer's cached slots; with a
        budget the slots' attention weights are accumulated. A sequence that reserved no token last
        gets zeros and accumulates nothing. Pages that neighbouring sequences share are read once where that
        saves ``shared_bytes``."""
        if self.groups is not None and self._shared_call_pays(window):
            return paged_shared_attention(q, self.k[layer], self.v[layer], self.page_table, self.queried,
                                          self._spans[:len(self._host_spans)], self.prefix, window=window)
        if self.budget is not None and self._provisional:
            for b in [b for b in self._provisional if self._grew[b]]:
                del self._provisional[b]  # its prompt is over
        return paged_attention(q, self.k[layer], self.v[layer], self.page_table, self.queried,
                               window=window,
                               weights=None if self.weights is None else self.weights[layer])

    def weigh(self, layer: int, q: torch.Tensor, lengths: torch.Tensor, *,
              provisional: Sequence[int] = ()) -> None:
        """Accumulates the attention weights of one query row per sequence over its first
        ``lengths[b]`` slots (int32 on the device; 0: none) in the layer's table, and nothing else. Those
        of ``provisional`` sequences can be taken back (:meth:`withdraw`) until they attend, an eviction
        goes by them or others are accumulated that cannot."""
        require(self.budget is not None, "this cache has no budget")
        if not provisional:
            self._provisional.clear()
        for b in provisional:
            self._provisional.setdefault(b, {})[layer] = self.weights[layer][b].clone()
        paged_attention(q, self.k[layer], self.v[layer], self.page_table, lengths,
                        weights=self.weights[layer])

    def withdraw(self, sequences: Sequence[int]) -> None:
        """Takes back the provisional weights of these sequences, where they have any."""
        require(self.budget is not None, "this cache has no budget")
        for b in sequences:
            for layer, before in self._provisional.pop(b, {}).items():
                self.weights[layer][b].copy_(before)

    def gather(self, layer: int, b: int):
        """(K, V) ``[H_kv, length, D]`` of sequence b, copied out of its pages."""
        n = self.host_lengths[b]
        pages = torch.tensor(self.host_pages[b], dtype=torch.int64, device=self.device)
        return tuple(x[pages].transpose(0, 1).flatten(1, 2)[:, :n] for x in (self.k[layer], self.v[layer]))

    def evict(self) -> None:
        """Brings every sequence down to the budget, in all layers, and frees the pages past it.
        Tokens reserved before it that are not appended yet have no slots any more."""
        require(self.budget is not None, "this cache has no budget")
        for i in range(len(self.k)):
            paged_evict(self.k[i], self.v[i], self.page_table, self.lengths, self.weights[i],
                        self.pos[i], self.seen, self.budget, sinks=self.sinks, recent=self.recent,
                        weights_out=self._spare_weights, pos_out=self._spare_pos)
            self.weights[i], self._spare_weights = self._spare_weights, self.weights[i]
            self.pos[i], self._spare_pos = self._spare_pos, self.pos[i]
        self._provisional.clear()
        if max(self.host_lengths) > self.budget:
            self._tokens = None
        changed = [b for b, n in enumerate(self.host_lengths)
                   if n > self.budget and self._resize(b, self.budget)]
        self._publish(changed)
