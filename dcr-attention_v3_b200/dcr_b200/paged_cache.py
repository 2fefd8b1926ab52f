"""A paged key-value cache for a batch of sequences and all layers of a model.

:class:`~dcr_b200.kv_cache.StaticKVCache` gives every sequence of a layer ``N_max`` positions from
the start; :class:`PagedKVCache` hands out pages of ``page_size`` slots as sequences grow, takes
them back when a sequence ends or its slots are evicted, and keeps one page table for all layers
(a page number means the same page of every layer's pool). With a ``budget`` it also keeps, per
layer, the accumulated attention weight and the position of every slot, and evicts what is over
the budget (``paged_evict``). The reference concatenates one contiguous cache per layer
(dcr_attention/models/llama/compat.py:208-254) and has no counterpart.

The host knows every length, so page handling never waits for the device; lengths, slots and
positions are also on the device, where the kernels read them.
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch

from dcr_b200.kernel.cuda._common import HEAD_DIM, check_dtype, require
from dcr_b200.kernel.cuda.paged import (PAGED_HEAD_DIMS, paged_append, paged_attention,
                                        paged_evict)


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
        self.weights = self.pos = None
        if budget is not None:
            tables = (batch, H_kv, self.max_pages * page_size)
            f32 = dict(dtype=torch.float32, device=self.device)
            self.weights = [torch.zeros(tables, **f32) for _ in range(layers)]
            self.pos = [torch.zeros(tables, **i32) for _ in range(layers)]
            self._spare_weights, self._spare_pos = torch.zeros(tables, **f32), torch.zeros(tables, **i32)
        self.free_pages = list(range(pages - 1, -1, -1))
        self.host_lengths = [0] * batch
        self.host_seen = [0] * batch
        self._grew = [False] * batch                 # the sequences that reserved a token last
        self.host_pages: List[List[int]] = [[] for _ in range(batch)]
        self._tokens = None  # (seq, slots, positions) of the tokens reserved last

    # ------------------------------------------------------------------------------- host side
    def _publish(self, rows: Sequence[int]) -> None:
        """Copies the host's lengths and the page table's given rows to the device."""
        pinned = self.device.type == "cuda"

        def to_device(dst, values):
            src = torch.tensor(values, dtype=torch.int32)
            dst.copy_(src.pin_memory() if pinned else src, non_blocking=pinned)
        to_device(self.lengths, self.host_lengths)
        to_device(self.seen, self.host_seen)
        to_device(self.queried, [n if g else 0 for n, g in zip(self.host_lengths, self._grew)])
        for b in rows:
            held = self.host_pages[b]
            to_device(self.page_table[b], held + [-1] * (self.max_pages - len(held)))

    def _resize(self, b: int, length: int) -> bool:
        """Gives sequence b the pages of `length` slots; True if they changed."""
        need, held = -(-length // self.page_size), self.host_pages[b]
        before = len(held)
        while len(held) < need:
            held.append(self.free_pages.pop())
        while len(held) > need:
            self.free_pages.append(held.pop())
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
        self._tokens = tuple(torch.tensor(x, **i32).to(self.device) for x in (seq, slots, positions))
        return len(seq)

    def release(self, b: int) -> None:
        """Ends sequence b: its pages go back to the pool."""
        self._resize(b, 0)
        self.host_seen[b], self._grew[b] = 0, False
        self._publish([b])

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

    def attend(self, layer: int, q: torch.Tensor, *, window: int = 0) -> torch.Tensor:
        """O ``[batch, H, D]`` of one query row per sequence over the layer's cached slots; with a
        budget the slots' attention weights are accumulated. A sequence that reserved no token last
        gets zeros and accumulates nothing."""
        return paged_attention(q, self.k[layer], self.v[layer], self.page_table, self.queried,
                               window=window,
                               weights=None if self.weights is None else self.weights[layer])

    def weigh(self, layer: int, q: torch.Tensor, lengths: torch.Tensor) -> None:
        """Accumulates the attention weights of one query row per sequence over its first
        ``lengths[b]`` slots (int32 on the device; 0: none) in the layer's table, and nothing else."""
        require(self.budget is not None, "this cache has no budget")
        paged_attention(q, self.k[layer], self.v[layer], self.page_table, lengths,
                        weights=self.weights[layer])

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
        if max(self.host_lengths) > self.budget:
            self._tokens = None
        changed = [b for b, n in enumerate(self.host_lengths)
                   if n > self.budget and self._resize(b, self.budget)]
        self._publish(changed)
