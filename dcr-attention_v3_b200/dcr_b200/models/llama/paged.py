"""Serving a Llama-architecture model from a paged cache: ragged prompts, decode steps, eviction
and processed logits.

:class:`PagedLlamaDecoder` runs the weights of a
:class:`~dcr_b200.models.llama.model.DCRLlamaDecoder` over a
:class:`~dcr_b200.paged_cache.PagedKVCache`: sequences of unequal lengths in one batch, a cache that
grows by pages and, with a budget, forgets the slots that drew the least attention. Per layer and
step: a norm, the q/k/v GEMM, query/key norms (``qk_norm``) with rotation and append in one launch,
attention over the pages, o_proj and the MLP. Prompts go in whole or in chunks, beside sequences that
run already, and on a common prefix that is computed and held once. :meth:`PagedLlamaDecoder.generate` is the loop around
it with penalties, bias and grammar masks on the logits. The reference decodes equal sequences
greedily over one contiguous cache (tests/kernel/test_m1_acceptance.py:198).
"""
from __future__ import annotations

from typing import Callable, List, Optional, Sequence

import torch
import torch.nn.functional as F

from dcr_b200.kernel.cuda._common import HEAD_DIM, require
from dcr_b200.kernel.cuda.decode_ops import add_rmsnorm, silu_mul_packed
from dcr_b200.kernel.cuda.logits import process_logits
from dcr_b200.models.llama.model import DCRLlamaDecoder
from dcr_b200.paged_cache import PagedKVCache


class PagedLlamaDecoder(torch.nn.Module):
    """``model``'s weights over paged caches. ``qk_norm``: every layer RMS-norms its query and key
    heads before the rotation, with its own weights ``q_norm[i]`` and ``k_norm[i]`` (ones at first;
    a checkpoint's go there). ``max_positions``: rows of the position tables. ``inv_freq`` (fp32 ``[r /
    2]``): rotate by these frequencies instead of the model's tables, with ``interleaved`` pairs and an
    amplitude ``rotary_factor`` if wanted (:func:`~dcr_b200.kernel.cuda.rotary.rotary`)."""

    def __init__(self, model: DCRLlamaDecoder, *, qk_norm: bool = False, max_positions: int = 32768,
                 inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False,
                 rotary_factor: float = 1.0):
        super().__init__()
        require(model.fast, "the paged decoder runs the packed projections of fast models")
        self.model, self.qk_norm = model, qk_norm
        kw = dict(dtype=model.dtype, device=model.device)
        norms = lambda: torch.nn.ParameterList(  # noqa: E731
            torch.nn.Parameter(torch.ones(HEAD_DIM, **kw)) for _ in model.layers if qk_norm)
        self.q_norm, self.k_norm = norms(), norms()
        self.cos, self.sin = (t.contiguous() for t in model.rope_table(max_positions))
        require(inv_freq is not None or (not interleaved and rotary_factor == 1.0),
                "interleaved pairs and an amplitude go with inv_freq")
        self.inv_freq = None if inv_freq is None else inv_freq.to(model.device, torch.float32).contiguous()
        self.interleaved, self.rotary_factor = interleaved, rotary_factor

    def new_cache(self, batch: int, pages: int, max_slots: int, **kw) -> PagedKVCache:
        """A cache for this model (keywords as :class:`PagedKVCache`)."""
        return PagedKVCache(len(self.model.layers), batch, self.model.cfg.kv_heads, pages, max_slots,
                            dtype=self.model.dtype, device=self.model.device, **kw)

    def _check_positions(self, cache: PagedKVCache, new_tokens: Sequence[int]) -> None:
        """Refuses, before the cache changes, tokens past the position table."""
        require(len(new_tokens) == cache.batch, f"{cache.batch} sequences expected")
        for b, n in enumerate(new_tokens):
            require(n == 0 or self.inv_freq is not None or cache.host_seen[b] + n <= self.cos.shape[0],
                    f"sequence {b} would reach position {cache.host_seen[b] + n} of a table of "
                    f"{self.cos.shape[0]}")

    def _layers(self, tokens: torch.Tensor, cache: PagedKVCache,
                attend: Callable[[int, torch.Tensor], torch.Tensor]) -> torch.Tensor:
        """The normed hidden states [T, hidden] of T reserved tokens."""
        cfg = self.model.cfg
        nq, nk = cfg.heads * HEAD_DIM, cfg.kv_heads * HEAD_DIM
        T = tokens.shape[0]
        h, delta = self.model.embed_tokens(tokens), None
        for i, layer in enumerate(self.model.layers):
            eps = layer.input_layernorm.eps
            h, x = add_rmsnorm(h, delta, layer.input_layernorm.weight, eps)
            qkv = F.linear(x, layer.self_attn._qkv)
            q = qkv[:, :nq].view(T, cfg.heads, HEAD_DIM)
            k = qkv[:, nq:nq + nk].view(T, cfg.kv_heads, HEAD_DIM)
            v = qkv[:, nq + nk:].view(T, cfg.kv_heads, HEAD_DIM)
            norms = dict(eps=eps, q_weight=self.q_norm[i] if self.qk_norm else None,
                         k_weight=self.k_norm[i] if self.qk_norm else None)
            if self.inv_freq is None:
                q = cache.append(i, q, k, v, self.cos, self.sin, **norms)
            else:
                q = cache.append_rotary(i, q, k, v, self.inv_freq, interleaved=self.interleaved,
                                        factor=self.rotary_factor, **norms)
            a = layer.self_attn.o_proj(attend(i, q).reshape(T, nq))
            h, x = add_rmsnorm(h, a, layer.post_attention_layernorm.weight, eps)
            delta = layer.down_proj(silu_mul_packed(F.linear(x, layer._gate_up)))
        return add_rmsnorm(h, delta, self.model.norm.weight, self.model.norm.eps)[1]

    @torch.no_grad()
    def prefill(self, prompts: Sequence[Sequence[int]], cache: PagedKVCache, *,
                prefix: Optional[Sequence[int]] = None) -> torch.Tensor:
        """Feeds the next tokens of each sequence (none: it stays idle) behind what the cache holds of
        it: whole prompts, or chunks of them, beside sequences that are further. Returns the logits
        [batch, vocab] after each one's last token (zeros for idle sequences). A ``prefix`` precedes
        every prompt of an empty cache: it is computed once, and its full pages are held once. In a
        cache with a budget, attention weights begin to accumulate with the decode steps; a sequence
        over the budget, which may be evicted before its next step attends, begins with those of its
        last token (of its prompt's last chunk, where no eviction comes between the chunks)."""
        require(len(prompts) == cache.batch, f"{cache.batch} prompts expected")
        lengths = [len(p) for p in prompts]
        require(sum(lengths) > 0, "at least one prompt must hold a token")
        vocab = self.model.cfg.vocab
        require(all(0 <= t < vocab for p in (*prompts, prefix or ()) for t in p),
                f"prompt ids must be in [0, {vocab})")
        if prefix:
            require(not any(cache.host_lengths), "a prefix expects an empty cache")
            require(cache.budget is None, "a cache with a budget shares no prefix")
            whole = [len(prefix) + n if n else 0 for n in lengths]
            self._check_positions(cache, whole)
            require(max(whole) <= cache.max_slots, f"{max(whole)} tokens in {cache.max_slots} slots")
            live = [b for b, n in enumerate(lengths) if n]
            shared = len(prefix) // cache.page_size * (len(live) - 1)
            pages = sum(-(-n // cache.page_size) for n in whole) - shared
            require(pages <= len(cache.free_pages), f"{pages} pages needed, {len(cache.free_pages)} free")
            self.prefill([prefix if b == live[0] else [] for b in range(cache.batch)], cache)
            cache.fork(live[0], live[1:])
        self._check_positions(cache, lengths)
        if cache.over_budget():
            cache.evict()
        cache.reserve(lengths)
        flat = torch.tensor([t for p in prompts for t in p], dtype=torch.int64).to(self.model.device)
        begins = [sum(lengths[:b]) for b in range(len(lengths))]
        over = last_rows = None
        provisional = []
        held = [h if n else 0 for h, n in zip(cache.host_lengths, lengths)]
        if cache.budget is not None:
            cache.withdraw([b for b, n in enumerate(lengths) if n])  # more of their prompts follows
        if cache.budget is not None and max(held) > cache.budget:
            if not cache.over_budget():  # else they are evicted next, with these weights
                provisional = [b for b, h in enumerate(held) if h > cache.budget]
            over = torch.tensor([h if h > cache.budget else 0 for h in held],
                                dtype=torch.int32).to(self.model.device)
            last_rows = torch.tensor([begins[b] + n - 1 if n else 0
                                      for b, n in enumerate(lengths)]).to(self.model.device)

        def attend(i, q):
            if over is not None:
                cache.weigh(i, q[last_rows], over, provisional=provisional)
            return cache.prefill_attend(i, q)

        x = self._layers(flat, cache, attend)
        logits = torch.zeros(cache.batch, self.model.cfg.vocab, dtype=x.dtype, device=x.device)
        live = [b for b, n in enumerate(lengths) if n]
        last = torch.tensor([begins[b] + lengths[b] - 1 for b in live], device=x.device)
        logits[torch.tensor(live, device=x.device)] = self.model.lm_head(x[last])
        return logits

    @torch.no_grad()
    def step(self, tokens: torch.Tensor, cache: PagedKVCache,
             active: Optional[Sequence[bool]] = None) -> torch.Tensor:
        """One decode step: appends ``tokens`` [batch] (ids on the device) and returns the logits
        [batch, vocab]. Sequences that are not ``active`` neither grow nor attend (their rows mean
        nothing). Evicts first where the cache is over its budget."""
        require(tokens.shape == (cache.batch,) and tokens.dtype in (torch.int64, torch.int32) and
                tokens.device == self.cos.device,
                f"tokens must be {cache.batch} ids on {self.cos.device}")
        live = [True] * cache.batch if active is None else [bool(a) for a in active]
        self._check_positions(cache, [int(a) for a in live])
        if cache.over_budget():
            cache.evict()
        T = cache.reserve([int(a) for a in live])
        if T == cache.batch:
            x = self._layers(tokens, cache, lambda i, q: cache.attend(i, q))
            return self.model.lm_head(x)
        rows = torch.tensor([b for b, a in enumerate(live) if a], dtype=torch.int64).to(self.model.device)

        def attend(i, q):  # the other sequences' rows ride along as zeros, and are dropped
            full = q.new_zeros(cache.batch, q.shape[1], q.shape[2])
            full[rows] = q
            return cache.attend(i, full)[rows]

        x = self._layers(tokens[rows], cache, attend)
        logits = torch.zeros(cache.batch, self.model.cfg.vocab, dtype=x.dtype, device=x.device)
        logits[rows] = self.model.lm_head(x)
        return logits

    @torch.no_grad()
    def generate(self, prompts: Sequence[Sequence[int]], cache: PagedKVCache, max_new: int, *,
                 repetition: Optional[torch.Tensor] = None,
                 presence: Optional[torch.Tensor] = None,
                 frequency: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                 allowed: Optional[Callable[[List[List[int]]], Optional[torch.Tensor]]] = None,
                 stop: Optional[int] = None, prefix: Optional[Sequence[int]] = None) -> List[List[int]]:
        """Greedy generation of up to ``max_new`` tokens after each prompt, which must not be empty;
        a ``prefix`` precedes all of them and is computed and held once (:meth:`prefill`).

        The penalties, ``bias`` and mask are those of
        :func:`~dcr_b200.kernel.cuda.logits.process_logits`; ``allowed(generated)`` returns a step's
        mask (or None). A sequence ends at the token ``stop`` (kept), or where its mask allows
        none; its pages are freed then."""
        require(len(prompts) == cache.batch, f"{cache.batch} prompts expected")
        require(max_new > 0 and all(len(p) > 0 for p in prompts), "prompts must hold a token each")
        B, dev = cache.batch, self.model.device
        whole = [[*(prefix or ()), *p] for p in prompts]
        width = max(len(p) for p in whole) + max_new
        history = torch.full((B, width), -1, dtype=torch.int64)
        for b, p in enumerate(whole):
            history[b, :len(p)] = torch.tensor(p, dtype=torch.int64)
        history = history.to(dev)
        n_prompt = torch.tensor([len(p) for p in whole], dtype=torch.int32).to(dev)
        n_tok = n_prompt.clone()
        out: List[List[int]] = [[] for _ in range(B)]
        live = [True] * B
        logits = self.prefill(prompts, cache, prefix=prefix)
        for i in range(max_new):
            mask = None if allowed is None else allowed(out)
            _, token = process_logits(logits, tokens=history, token_lengths=n_tok,
                                      prompt_lengths=n_prompt, repetition=repetition,
                                      presence=presence, frequency=frequency, bias=bias,
                                      allowed=mask, out=logits)
            history.scatter_(1, n_tok.long()[:, None], token[:, None])
            n_tok += 1
            for b, t in enumerate(token.tolist()):
                if not live[b]:
                    continue
                if t >= 0:
                    out[b].append(t)
                if t < 0 or t == stop:
                    live[b] = False
                    cache.release(b)
            if not any(live) or i + 1 == max_new:
                break
            logits = self.step(token.clamp(min=0), cache, live)
        for b in range(B):
            if live[b]:
                cache.release(b)
        return out
