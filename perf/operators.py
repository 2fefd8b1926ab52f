"""The paged serving operators, as measured cases: what goes in, a plain form in elementary torch
operations, the framework's own calls, the work that cannot be avoided, and a 64-bit definition.

Four operators of one decode step over a paged key-value cache:

* ``attend``: attention of one new token per sequence over the pages of its cache; optionally it
  also adds each slot's attention weight (summed over the query heads of a KV head) to a running
  table.
* ``append``: RMS norms of every query and key head with the position rotation, and the new keys
  and values written into their pages.
* ``evict``: keeps a budget of slots per sequence and KV head by the accumulated attention weight
  (first and most recent positions always), and moves the kept rows into the first slots.
* ``logits``: penalties for repeated tokens, a bias and a grammar mask on the logits, and the
  greedy token.

Heads follow Llama-3.2-1B's layout (32 query heads on 8 KV heads of 64, vocabulary 128256) where
a case does not say otherwise; 32768 positions and a kept share of 15% are the context and the
coverage that this repository's decode step is measured at.
"""
import math

import torch

own = False  # False: the plain forms below; True: the framework's operators

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------------------------- the cases
def _attend(name, B, H, H_kv, D, n, page, dtype, ragged=False, window=0, weights=False):
    c = {"op": "attend", "B": B, "H": H, "H_kv": H_kv, "D": D, "n": n, "page": page,
         "dtype": dtype, "ragged": ragged, "window": window, "weights": weights}
    return dict(c, name=name) if name else c


def _append(name, T, H, H_kv, D, page, dtype, prompt=False, table=True):
    c = {"op": "append", "T": T, "H": H, "H_kv": H_kv, "D": D, "page": page, "dtype": dtype,
         "prompt": prompt, "table": table}
    return dict(c, name=name) if name else c


def _evict(name, B, H_kv, D, n, budget, sinks, recent, page, dtype, ragged=False):
    c = {"op": "evict", "B": B, "H_kv": H_kv, "D": D, "n": n, "budget": budget, "sinks": sinks,
         "recent": recent, "page": page, "dtype": dtype, "ragged": ragged}
    return dict(c, name=name) if name else c


def _logits(name, B, V, L, dtype, bias, mask):
    c = {"op": "logits", "B": B, "V": V, "L": L, "dtype": dtype, "bias": bias, "mask": mask}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user, a short conversation: the smallest call, latency counts
        _attend("attend one short", 1, 32, 8, 64, 1000, 16, "bf16"),
        # the batch and context that the decode step is measured at, one token past them
        _attend("attend long context", 4, 32, 8, 64, 32769, 64, "bf16"),
        # a serving batch of unequal sequences, some of them finished (length 0)
        _attend("attend ragged batch", 48, 32, 8, 64, 16000, 16, "f16", ragged=True),
        # heads of 128, eight query heads on a KV head, a sliding window that begins inside a page
        _attend("attend window heads of 128", 16, 64, 8, 128, 20011, 32, "bf16", window=8191),
        # single precision, one query head per KV head
        _attend("attend single precision", 3, 16, 16, 64, 8195, 16, "f32"),
        # a step of a cache under eviction: the weights of all slots are accumulated
        _attend("attend with weights", 8, 32, 8, 64, 16385, 64, "bf16", weights=True),
        # one decode step of a batch: a new token per sequence
        _append("append one step", 48, 32, 8, 64, 16, "bf16"),
        # prompts of several sequences, heads of 128
        _append("append prompts", 16381, 32, 8, 128, 64, "f16", prompt=True),
        # steady state: one slot over the budget, one goes
        _evict("evict one", 8, 8, 64, 4917, 4916, 4, 256, 64, "bf16"),
        # after a long prompt: 15% of 32768 positions stay
        _evict("evict long prompt", 4, 8, 64, 32768, 4916, 4, 512, 64, "bf16"),
        # one user: the LM head's row, a conversation of a thousand tokens
        _logits("logits one", 1, 128256, 1000, "bf16", False, False),
        # a serving batch with a bias for the vocabulary and a grammar mask for each row
        _logits("logits batch", 128, 128256, 8192, "f32", True, True),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("attend", "attend", "append", "evict", "logits"))
    D = rng.choice((64, 64, 128))
    page = rng.choice((8, 16, 32, 48, 64, 128))
    if op == "attend":
        H_kv = rng.choice((1, 2, 4, 8, 16))
        G = rng.choice((1, 2, 3, 4, 5, 7, 8, 12, 16))
        dtype = rng.choice(("bf16", "f16", "f32"))
        B = _log_uniform(rng, 1, 96)
        # no more bytes than the largest listed attention reads
        most = 800_000_000 // (B * H_kv * D * BYTES[dtype] * 2)
        n = _log_uniform(rng, 1, max(1, min(131072, most)))
        return _attend(None, B, G * H_kv, H_kv, D, n, page, dtype, ragged=rng.random() < 0.5,
                       window=rng.choice((0, 0, _log_uniform(rng, 1, 8192))),
                       weights=rng.random() < 0.3)
    if op == "append":
        H_kv = rng.choice((1, 2, 4, 8))
        G = rng.choice((1, 2, 3, 4, 5, 8))
        return _append(None, _log_uniform(rng, 1, 8192), G * H_kv, H_kv, D, page,
                       rng.choice(("bf16", "f16", "f32")), prompt=rng.random() < 0.5,
                       table=rng.random() < 0.7)
    if op == "evict":
        H_kv = rng.choice((1, 2, 4, 8))
        B = _log_uniform(rng, 1, 32)
        n = _log_uniform(rng, 2, min(65536, 1048576 // (B * H_kv)))
        budget = max(1, min(n, int(n * rng.choice((0.05, 0.15, 0.5, 0.9, 1.0)))))
        return _evict(None, B, H_kv, D, n, budget, rng.choice((0, 1, 4)),
                      rng.choice((0, 1, budget // 8, budget // 2)), page,
                      rng.choice(("bf16", "f16", "f32")), ragged=rng.random() < 0.5)
    V = _log_uniform(rng, 1000, 200000)
    B = _log_uniform(rng, 1, min(128, 12_000_000 // V + 1))
    return _logits(None, B, V, _log_uniform(rng, 1, 8192), rng.choice(("bf16", "f16", "f32")),
                   rng.random() < 0.5, rng.random() < 0.5)


# ------------------------------------------------------------------- lengths that a case stands for
def _lengths(case):
    """Each sequence's number of cached slots: n, or spread over [0, n], a fixed rule of the case."""
    B, n = case["B"], case["n"]
    if not case["ragged"]:
        return [n] * B
    # the golden-ratio sequence spreads evenly; its first member is the longest, one in 16 is empty
    return [n if b == 0 else 0 if b % 16 == 9 else max(1, int(n * ((b * 0.6180339887498949) % 1.0)))
            for b in range(B)]


def _prompts(T):
    """Prompt lengths of a ragged prefill of T tokens: shares of 1, 2, 3, ... of what is left."""
    out, left, k = [], T, 2
    while left > 0:
        n = max(1, left // k) if len(out) < 7 else left
        out.append(n)
        left -= n
        k = 2 if k == 3 else 3
    return out


# ---------------------------------------------------------------------------------------- the inputs
def _pool(g, lengths, H_kv, page, D, dt, dev, fill):
    """Pages of all sequences in a scattered order: (k_pages, v_pages, page_table). Slots that no
    token was written to hold NaN, as memory that was never written may."""
    need = [(n + page - 1) // page for n in lengths]
    width = max(max(need), 1)
    total = max(sum(need), 1)
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    flat = torch.full((len(lengths), width), -1, dtype=torch.int32)
    used = 0
    rows, cols = [], []
    for b, m in enumerate(need):
        rows += [b] * m
        cols += range(m)
        used += m
    table = flat.to(dev)
    if used:
        table[torch.tensor(rows, device=dev), torch.tensor(cols, device=dev)] = order[:used]
    shape = (total, H_kv, page, D)
    if not fill:
        return torch.zeros(shape, dtype=dt, device=dev), torch.zeros(shape, dtype=dt, device=dev), table
    k = torch.randn(shape, generator=g, device=dev, dtype=torch.float32 if dt == torch.float32 else dt)
    v = torch.randn(shape, generator=g, device=dev, dtype=k.dtype)
    for b, (n, m) in enumerate(zip(lengths, need)):
        if n:
            k[table[b, 0].long(), :, :4] *= 4.0  # the first positions draw much attention
            if n % page:
                last = table[b, m - 1].long()
                k[last, :, n % page:] = float("nan")
                v[last, :, n % page:] = float("nan")
    return k, v, table


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    op = case["op"]
    s = {"case": case}
    if op == "attend":
        dt = DTYPES[case["dtype"]]
        lengths = _lengths(case)
        s["k_pages"], s["v_pages"], s["table"] = _pool(g, lengths, case["H_kv"], case["page"],
                                                       case["D"], dt, dev, True)
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
        s["q"] = torch.randn(case["B"], case["H"], case["D"], generator=g, device=dev).to(dt)
        if case["weights"]:
            cap = s["table"].shape[1] * case["page"]
            # what some steps have left there: about each query head's share of 1 a slot and step
            share = case["H"] / case["H_kv"] / case["n"]
            s["weights"] = share * torch.rand(case["B"], case["H_kv"], cap, generator=g, device=dev)
    elif op == "append":
        dt = DTYPES[case["dtype"]]
        T, H, H_kv, D, page = (case[x] for x in ("T", "H", "H_kv", "D", "page"))
        if case["prompt"]:
            parts = _prompts(T)
            seq = [b for b, n in enumerate(parts) for _ in range(n)]
            slot = [i for n in parts for i in range(n)]
            lengths, position = parts, slot
        else:  # sequences that already hold some slots; positions run ahead of them (evicted slots)
            seq = list(range(T))
            slot = [(7 * b + 3) % page for b in range(T)]
            lengths = [page] * T
            position = [x + 37 * b % 4096 for b, x in enumerate(slot)]
        s["k_pages"], s["v_pages"], s["page_table"] = _pool(g, lengths, H_kv, page, D, dt, dev, False)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        s["seq"], s["slots"], s["positions"] = i32(seq), i32(slot), i32(position)
        # one row of the packed projections per token; q, k and v are slices of it
        s["qkv"] = torch.randn(T, (H + 2 * H_kv) * D, generator=g, device=dev).to(dt)
        s["qw"] = (1.0 + 0.2 * torch.randn(D, generator=g, device=dev)).to(dt)
        s["kw"] = (1.0 + 0.2 * torch.randn(D, generator=g, device=dev)).to(dt)
        inv = 500000.0 ** (-torch.arange(0, D, 2, device=dev).double() / D)
        angle = torch.arange(max(position) + 1, device=dev).double()[:, None] * inv
        angle = torch.cat((angle, angle), dim=1)
        s["cos"], s["sin"] = angle.cos().to(dt), angle.sin().to(dt)
        if case["table"]:  # a cache under eviction: a slot's weight begins at 0, its position is kept
            cap = s["page_table"].shape[1] * page
            s["weights"] = torch.rand(len(lengths), H_kv, cap, generator=g, device=dev)
            s["pos"] = torch.zeros(len(lengths), H_kv, cap, dtype=torch.int32, device=dev)
    elif op == "evict":
        dt = DTYPES[case["dtype"]]
        B, H_kv = case["B"], case["H_kv"]
        lengths = _lengths(case)
        s["k_pages"], s["v_pages"], s["table"] = _pool(g, lengths, H_kv, case["page"], case["D"],
                                                       dt, dev, True)
        cap = s["table"].shape[1] * case["page"]
        # attention weight: few slots have much of it, many have little, some have none at all
        u = torch.rand(B, H_kv, cap, generator=g, device=dev)
        w = (1.0 / (u + 1e-3)) * (torch.rand(B, H_kv, cap, generator=g, device=dev) > 0.05)
        s["weights"] = w.contiguous()
        # slots of an evicted cache are in no order: positions are a permutation for each head
        gap = 3
        s["pos"] = (gap * torch.rand(B, H_kv, cap, generator=g, device=dev).argsort(-1)).to(torch.int32)
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
        s["seen"] = torch.full((B,), gap * cap, dtype=torch.int32, device=dev)
    else:
        B, V, L = case["B"], case["V"], case["L"]
        s["logits"] = (4.0 * torch.randn(B, V, generator=g, device=dev)).to(DTYPES[case["dtype"]])
        # words repeat: the squared uniform favours low token ids
        u = torch.rand(B, L, generator=g, device=dev)
        s["tokens"] = (u * u * V).to(torch.int32).clamp_(max=V - 1)
        n = torch.tensor([max(0, L - (b * L) // (2 * B)) for b in range(B)], dtype=torch.int32, device=dev)
        s["token_lengths"], s["prompt_lengths"] = n, n // 3
        r = lambda lo, hi: lo + (hi - lo) * torch.rand(B, generator=g, device=dev)  # noqa: E731
        s["repetition"], s["presence"], s["frequency"] = r(1.0, 1.5), r(0.0, 1.0), r(0.0, 0.5)
        s["bias"] = torch.randn(V, generator=g, device=dev) if case["bias"] else None
        s["allowed"] = None
        if case["mask"]:  # some rows are free, the others may go on with a tenth or so of the tokens
            words = torch.randint(-2**31, 2**31, (3, B, (V + 31) // 32), generator=g, device=dev)
            word = words[0] & words[1] & words[2]
            word[::4] = -1
            s["allowed"] = word.to(torch.int32)
    return s


# -------------------------------------------------------------------------------- the plain forms
def _slots_of(pages, table):
    """[B, H_kv, slots, ...] in 32 bits of pages [pages, H_kv, page, ...] through a table [B, m]."""
    x = pages[table.clamp(min=0).long()].float()
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attend(s):
    c = s["case"]
    B, H, H_kv, D = c["B"], c["H"], c["H_kv"], c["D"]
    k, v = _slots_of(s["k_pages"], s["table"]), _slots_of(s["v_pages"], s["table"])
    at = torch.arange(k.shape[2], device=k.device)
    n = s["lengths"].long()[:, None]
    valid = (at < n) & (at >= n - c["window"] if c["window"] else at >= 0)
    valid &= (s["table"] >= 0).repeat_interleave(c["page"], 1)
    q = s["q"].float().view(B, H_kv, H // H_kv, D)
    score = (q @ k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    score = torch.where(valid[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    v = torch.where(valid[:, None, :, None], v, 0.0)
    out = {"o": (p @ v).view(B, H, D).to(s["q"].dtype), "lse": (torch.log(total) + top).view(B, H)}
    if c["weights"]:
        s["weights"] += p.sum(2)
        out["weights"] = s["weights"]
    return out


def _plain_append(s):
    c = s["case"]
    T, H, H_kv, D, page = (c[x] for x in ("T", "H", "H_kv", "D", "page"))
    dt = s["qkv"].dtype
    x = s["qkv"].float().view(T, H + 2 * H_kv, D)
    cos, sin = s["cos"].float()[s["positions"].long()], s["sin"].float()[s["positions"].long()]

    def turned(y, w):
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-5) * w.float()
        half = torch.cat((-y[..., D // 2:], y[..., :D // 2]), -1)
        return (y * cos[:, None] + half * sin[:, None]).to(dt)

    q, k = turned(x[:, :H], s["qw"]), turned(x[:, H:H + H_kv], s["kw"])
    slot, seq = s["slots"].long(), s["seq"].long()
    to = s["page_table"][seq, slot // page].long()
    s["k_pages"][to, :, slot % page] = k
    s["v_pages"][to, :, slot % page] = x[:, H + H_kv:].to(dt)
    out = {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if c["table"]:
        s["weights"][seq, :, slot] = 0.0
        s["pos"][seq, :, slot] = s["positions"][:, None].expand(T, H_kv)
        out.update(weights=s["weights"], pos=s["pos"])
    return out


def _plain_evict(s):
    c = s["case"]
    B, H_kv, page, budget = c["B"], c["H_kv"], c["page"], c["budget"]
    w, pos, n = s["weights"], s["pos"], s["lengths"].long()[:, None, None]
    cap = w.shape[2]
    at = torch.arange(cap, device=w.device).expand(B, H_kv, cap)
    first = (pos < c["sinks"]) | (pos >= (s["seen"] - c["recent"])[:, None, None])
    rank = torch.where(first, math.inf, w)
    rank = torch.where(at < n, rank, -math.inf)
    order = torch.argsort(rank, dim=-1, descending=True, stable=True)
    keep = torch.zeros_like(first).scatter_(2, order[..., :min(budget, cap)], True) & (at < n)
    # a kept slot past the budget goes to a free one before it: i-th to i-th, in slot order
    free = ~keep & (at < budget) & (at < n)
    move = keep & (at >= budget)
    movers = torch.sort(torch.where(move, at, cap), -1).values
    nth = (free.cumsum(-1) - 1).clamp(min=0)
    src = torch.where(free, movers.gather(2, nth), at)
    if cap < budget:
        src = torch.cat((src, src.new_full((B, H_kv, budget - cap), cap)), 2)
    src = src[..., :budget]
    held = torch.arange(budget, device=w.device) < n
    safe = src.clamp(max=cap - 1)
    src = torch.where(held, src, -1)
    w_out = torch.where(held, w.gather(2, safe), 0.0)
    pos_out = torch.where(held, pos.gather(2, safe), -1)
    # the rows: through the table, each head's own slots
    b, h, i = torch.nonzero(held & (src != torch.arange(budget, device=w.device)), as_tuple=True)
    f = src[b, h, i]
    fp, tp = s["table"][b, f // page].long(), s["table"][b, i // page].long()
    for pages in (s["k_pages"], s["v_pages"]):
        pages[tp, h, i % page] = pages[fp, h, f % page]
    return {"src": src.to(torch.int32), "weights": w_out, "pos": pos_out,
            "lengths": s["lengths"].clamp(max=budget), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_logits(s):
    c = s["case"]
    B, V, L = c["B"], c["V"], c["L"]
    x = s["logits"].float()
    at = torch.arange(L, device=x.device)
    held = at < s["token_lengths"][:, None]
    said = held & (at >= s["prompt_lengths"][:, None])
    tok = s["tokens"].long()
    zero = torch.zeros(B, V, device=x.device)
    seen = zero.scatter_add(1, tok, held.float()) > 0
    count = zero.scatter_add(1, tok, said.float())
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - count * s["frequency"][:, None]
    x = x - (count > 0).float() * s["presence"][:, None]
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["allowed"] is not None:
        bit = torch.arange(32, device=x.device, dtype=torch.int32)
        ok = ((s["allowed"][:, :, None] >> bit) & 1).view(B, -1)[:, :V].bool()
        x = torch.where(ok, x, -math.inf)
    x = x.to(s["logits"].dtype)
    token = x.float().argmax(-1)
    if s["allowed"] is not None:
        token = torch.where(ok.any(-1), token, -1)
    return {"logits": x, "token": token}


PLAIN = {"attend": _plain_attend, "append": _plain_append, "evict": _plain_evict,
         "logits": _plain_logits}


# ------------------------------------------------------------------------- the framework's operators
_calls = {}


def _framework():
    """The package's operators; its source root is put on the path as its users do."""
    if not _calls:
        import os
        import sys
        sys.path.insert(0, os.path.join(os.getcwd(), "dcr-attention_v3_b200"))
        from dcr_b200.kernel.cuda import logits, paged
        _calls.update(attend=paged.paged_attention, append=paged.paged_append,
                      evict=paged.paged_evict, logits=logits.process_logits)
    return _calls


def _own(s):
    c = s["case"]
    op = c["op"]
    call = _framework()[op]
    if op == "attend":
        o, lse = call(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"],
                      window=c["window"], weights=s.get("weights"), return_lse=True)
        out = {"o": o, "lse": lse}
        if c["weights"]:
            out["weights"] = s["weights"]
        return out
    if op == "append":
        H, H_kv, D = c["H"], c["H_kv"], c["D"]
        heads = s["qkv"].view(-1, H + 2 * H_kv, D)
        q = call(heads[:, :H], heads[:, H:H + H_kv], heads[:, H + H_kv:], s["cos"], s["sin"],
                 s["positions"], s["k_pages"], s["v_pages"], s["page_table"], s["slots"],
                 seq=s["seq"], q_weight=s["qw"], k_weight=s["kw"], eps=1e-5,
                 weights=s.get("weights"), pos=s.get("pos"))
        out = {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if c["table"]:
            out.update(weights=s["weights"], pos=s["pos"])
        return out
    if op == "evict":
        src, weights, pos, lengths = call(s["k_pages"], s["v_pages"], s["table"], s["lengths"],
                                          s["weights"], s["pos"], s["seen"], c["budget"],
                                          sinks=c["sinks"], recent=c["recent"])
        return {"src": src, "weights": weights, "pos": pos, "lengths": lengths,
                "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    x, token = call(s["logits"], tokens=s["tokens"], token_lengths=s["token_lengths"],
                    prompt_lengths=s["prompt_lengths"], repetition=s["repetition"],
                    presence=s["presence"], frequency=s["frequency"], bias=s["bias"],
                    allowed=s["allowed"])
    return {"logits": x, "token": token}


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------------------ the work of one pass
def work(case):
    op = case["op"]
    if op == "logits":
        B, V, L = case["B"], case["V"], case["L"]
        held = sum(max(0, L - (b * L) // (2 * B)) for b in range(B))
        b = 2 * B * V * BYTES[case["dtype"]] + 4 * held + 8 * B
        b += 4 * V if case["bias"] else 0
        b += B * ((V + 31) // 32) * 4 if case["mask"] else 0
        return {"bytes": b, "flops": 4 * B * V}
    H_kv, D, e = case["H_kv"], case["D"], BYTES[case["dtype"]]
    if op == "append":
        rows = case["T"] * (case["H"] + 2 * H_kv)
        b = 2 * rows * D * e + 12 * case["T"] + (8 * case["T"] * H_kv if case["table"] else 0)
        return {"bytes": b, "flops": 10 * case["T"] * (case["H"] + H_kv) * D}
    lengths = _lengths(case)
    if op == "attend":
        H, B = case["H"], case["B"]
        seen = [min(n, case["window"]) if case["window"] else n for n in lengths]
        b = sum(seen) * H_kv * D * e * 2 + 2 * B * H * D * e + 4 * B * H
        b += sum(4 * -(-n // case["page"]) for n in seen)
        b += 8 * sum(seen) * H_kv if case["weights"] else 0
        return {"bytes": b, "flops": 4 * sum(seen) * H * D}
    budget = case["budget"]
    b = 0.0
    for n in lengths:
        kept = min(n, budget)
        moved = kept * max(0, n - budget) / max(1, n)  # kept slots past the budget, on average
        b += H_kv * (8 * n + 12 * budget + 4 * moved * D * e)
    return {"bytes": b, "flops": H_kv * sum(lengths)}


# ------------------------------------------------------------- the definitions, evaluated in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "evict": _exact_evict,
            "logits": _exact_logits}[case["op"]](case, s)


def _exact_attend(c, s):
    B, H, H_kv, D, page = (c[x] for x in ("B", "H", "H_kv", "D", "page"))
    dev = s["q"].device
    o = torch.zeros(B, H, D, dtype=torch.float64, device=dev)
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device=dev)
    weights = s["weights"].double() if c["weights"] else None
    for b, n in enumerate(s["lengths"].tolist()):
        lo = max(0, n - c["window"]) if c["window"] else 0
        at = torch.arange(lo, n, device=dev)
        if not len(at):
            continue
        pg = s["table"][b, at // page].long()
        for h in range(H_kv):
            k = s["k_pages"][pg, h, at % page].double()
            v = s["v_pages"][pg, h, at % page].double()
            g = slice(h * (H // H_kv), (h + 1) * (H // H_kv))
            z = s["q"][b, g].double() @ k.T / math.sqrt(D)
            lse[b, g] = torch.logsumexp(z, -1)
            p = torch.softmax(z, -1)
            o[b, g] = p @ v
            if weights is not None:
                weights[b, h, lo:n] += p.sum(0)
    out = {"o": o, "lse": lse}
    if weights is not None:
        out["weights"] = weights
    return out


def _exact_append(c, s):
    T, H, H_kv, D, page = (c[x] for x in ("T", "H", "H_kv", "D", "page"))
    x = s["qkv"].double().view(T, H + 2 * H_kv, D)
    d = D // 2
    co, si = s["cos"].double()[s["positions"].long()], s["sin"].double()[s["positions"].long()]

    def one(y, w):
        y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / D + 1e-5) * w.double()
        a, b = y[..., :d], y[..., d:]
        return torch.cat((a * co[:, None, :d] - b * si[:, None, :d],
                          b * co[:, None, d:] + a * si[:, None, d:]), -1)

    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    slot, seq = s["slots"].long(), s["seq"].long()
    pg = s["page_table"][seq, slot // page].long()
    kp[pg, :, slot % page] = one(x[:, H:H + H_kv], s["kw"])
    vp[pg, :, slot % page] = x[:, H + H_kv:]
    out = {"q": one(x[:, :H], s["qw"]), "k_pages": kp, "v_pages": vp}
    if c["table"]:
        w = s["weights"].double()
        w[seq, :, slot] = 0.0
        out.update(weights=w, pos=None)
    return out


def _exact_evict(c, s):
    """Slot by slot on the host."""
    B, H_kv, page, budget = c["B"], c["H_kv"], c["page"], c["budget"]
    w, pos = s["weights"].double().cpu(), s["pos"].cpu()
    lengths, seen, table = s["lengths"].tolist(), s["seen"].tolist(), s["table"].tolist()
    w_out = torch.zeros(B, H_kv, budget, dtype=torch.float64)
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    fr, to = [], []
    for b in range(B):
        n = lengths[b]
        for h in range(H_kv):
            ws, ps = w[b, h, :n].tolist(), pos[b, h, :n].tolist()
            sure = [p < c["sinks"] or p >= seen[b] - c["recent"] for p in ps]
            kept = set(sorted(range(n), key=lambda i: (not sure[i], -ws[i] if not sure[i] else 0.0, i))[:budget])
            late = iter([i for i in range(budget, n) if i in kept])
            m = min(n, budget)
            src = [i if i in kept else next(late) for i in range(m)]
            if m:
                w_out[b, h, :m] = w[b, h, src]
            for i, j in enumerate(src):
                if i != j:
                    fr.append((table[b][j // page], h, j % page))
                    to.append((table[b][i // page], h, i % page))
    if fr:
        f, t = torch.tensor(fr, device=kp.device).T, torch.tensor(to, device=kp.device).T
        for pages in (kp, vp):
            pages[t[0], t[1], t[2]] = pages[f[0], f[1], f[2]]
    return {"src": None, "weights": w_out, "pos": None, "lengths": None, "k_pages": kp, "v_pages": vp}


def _exact_logits(c, s):
    V = c["V"]
    x = s["logits"].double()
    for b, (n, p) in enumerate(zip(s["token_lengths"].tolist(), s["prompt_lengths"].tolist())):
        all_ = torch.bincount(s["tokens"][b, :n].long(), minlength=V)
        new = torch.bincount(s["tokens"][b, p:n].long(), minlength=V).double()
        r = s["repetition"][b].double()
        y = torch.where(all_ > 0, torch.where(x[b] > 0, x[b] / r, x[b] * r), x[b])
        x[b] = y - new * s["frequency"][b].double() - (new > 0) * s["presence"][b].double()
    if s["bias"] is not None:
        x = x + s["bias"].double()
    if s["allowed"] is not None:
        t = torch.arange(V, device=x.device)
        x = x.masked_fill(((s["allowed"].long()[:, t // 32] >> (t % 32)) & 1) == 0, -math.inf)
    return {"logits": x, "token": None}
