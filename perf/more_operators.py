"""Prompts, shared prefixes and rotations over a paged cache, as measured cases: what goes in, a plain
form in elementary torch operations, the framework's own calls, the work that cannot be avoided, and
a 64-bit definition.

* ``prefill``: attention of many new tokens per sequence over the pages of its cache (a prompt, a chunk
  of one on a cached history, a few drafted tokens to verify), causal, optionally in a window.
* ``shared``: attention of one new token per sequence where groups of sequences hold the same pages
  in their first slots, which are read once for the group.
* ``rotary``: position rotation of query and key heads from frequencies, halves or neighbours paired,
  of the whole head or its first part, with a scaled amplitude.
* ``append``: that rotation with the query and key norms and the append into the pages.

Heads follow Llama-3.2-1B's layout (32 query heads on 8 KV heads of 64) where a case does not say
otherwise; 32768 positions is the context that this repository's decode step is measured at.
"""
import math

import torch

own = False  # False: the plain forms below; True: the framework's operators

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------------------------- the cases
def _prefill(name, B, n, history, H, H_kv, D, page, dtype, ragged=False, window=0):
    c = {"op": "prefill", "B": B, "n": n, "history": history, "H": H, "H_kv": H_kv, "D": D,
         "page": page, "dtype": dtype, "ragged": ragged, "window": window}
    return dict(c, name=name) if name else c


def _shared(name, B, groups, prefix, own_slots, H, H_kv, D, page, dtype, window=0):
    c = {"op": "shared", "B": B, "groups": groups, "prefix": prefix, "own": own_slots, "H": H,
         "H_kv": H_kv, "D": D, "page": page, "dtype": dtype, "window": window}
    return dict(c, name=name) if name else c


def _rotary(name, T, H, H_kv, D, rot, dtype, interleaved, in_place, far):
    c = {"op": "rotary", "T": T, "H": H, "H_kv": H_kv, "D": D, "rot": rot, "dtype": dtype,
         "interleaved": interleaved, "in_place": in_place, "far": far}
    return dict(c, name=name) if name else c


def _append(name, T, H, H_kv, D, rot, page, dtype, interleaved, norm, prompt, far):
    c = {"op": "append", "T": T, "H": H, "H_kv": H_kv, "D": D, "rot": rot, "page": page, "dtype": dtype,
         "interleaved": interleaved, "norm": norm, "prompt": prompt, "far": far}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user's question: the smallest prompt, latency counts
        _prefill("prefill one short", 1, 77, 0, 32, 8, 64, 16, "bf16"),
        # prompts of a batch, unequal, the longest of 8192 tokens
        _prefill("prefill ragged prompts", 6, 8192, 0, 32, 8, 64, 64, "bf16", ragged=True),
        # a chunk of a long document behind what is cached of it, heads of 128
        _prefill("prefill chunk on a long history", 1, 2048, 32768, 32, 8, 128, 64, "f16"),
        # drafted tokens of a serving batch, verified at once; a sliding window; some rows are idle
        _prefill("prefill drafted tokens", 48, 5, 16000, 32, 8, 64, 16, "f16", ragged=True, window=8191),
        # single precision, one query head per KV head
        _prefill("prefill single precision", 3, 999, 500, 16, 16, 64, 16, "f32", ragged=True),
        # a few samples of one short prompt
        _shared("shared short", 4, 1, 1008, 40, 32, 8, 64, 16, "bf16"),
        # a serving batch behind one system prompt, each at its own place in its answer
        _shared("shared system prompt", 64, 1, 8192, 700, 32, 8, 64, 64, "bf16"),
        # samples of several long documents, heads of 128, eight query heads on a KV head
        _shared("shared documents", 45, 3, 32768, 1500, 64, 8, 128, 32, "f16"),
        # one decode step of a batch: neighbours paired, half of the head, in place
        _rotary("rotary one step", 48, 32, 8, 64, 32, "bf16", True, True, 131072),
        # a prompt, halves paired, whole heads of 128, positions past a million
        _rotary("rotary long prompt", 16381, 32, 8, 128, 128, "f16", False, False, 1048576),
        # one decode step of a batch with norms
        _append("append one step", 48, 32, 8, 64, 64, 16, "bf16", False, True, False, 131072),
        # prompts, three quarters of each head, neighbours paired
        _append("append prompts", 16381, 32, 8, 128, 96, 64, "bf16", True, True, True, 131072),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("prefill", "prefill", "shared", "shared", "rotary", "append"))
    dtype = rng.choice(("bf16", "f16", "bf16", "f16", "f32"))
    D = rng.choice((64, 64, 128))
    page = rng.choice((8, 16, 24, 32, 64, 128))
    H_kv = rng.choice((1, 2, 4, 8))
    G = rng.choice((1, 2, 3, 4, 5, 8, 16))
    if op == "prefill":
        B = _log_uniform(rng, 1, 64)
        # no more arithmetic than the largest listed prefill, or than a pass in 32 bits bears
        most = 4e10 if dtype == "f32" else 8e11
        n = _log_uniform(rng, 1, 8192)
        history = rng.choice((0, _log_uniform(rng, 1, 32768)))
        while 4 * D * G * H_kv * B * n * (history + n) > most:
            B, n, history = max(1, B // 2), max(1, int(n / 1.5)), int(history / 1.2)
        return _prefill(None, B, n, history, G * H_kv, H_kv, D, page, dtype, ragged=rng.random() < 0.6,
                        window=rng.choice((0, 0, _log_uniform(rng, 1, 8192))))
    if op == "shared":
        B = _log_uniform(rng, 1, 96)
        groups = rng.randint(1, max(1, min(B, 6)))
        prefix = _log_uniform(rng, 1, 32768)
        own_slots = _log_uniform(rng, 1, 2000)
        most = 100_000_000 if dtype == "f32" else 400_000_000
        while 2 * D * H_kv * BYTES[dtype] * (groups * prefix + B * own_slots) > most:
            prefix, own_slots = max(1, prefix // 2), max(1, own_slots // 2)
        return _shared(None, B, groups, prefix, own_slots, G * H_kv, H_kv, D, page, dtype,
                       window=rng.choice((0, 0, 0, _log_uniform(rng, 1, 20000))))
    T = _log_uniform(rng, 1, 8192)
    far = rng.choice((4096, 131072, 1048576))
    H = min(G * H_kv, 64)
    H -= H % H_kv
    if op == "rotary":
        D = rng.choice((64, 80, 96, 128, 256))
        rot = rng.choice((D, D // 2, D // 4, 16))
        return _rotary(None, T, H, H_kv, D, rot, dtype, rng.random() < 0.5, rng.random() < 0.5, far)
    rot = rng.choice((D, D // 2, D // 4, 3 * D // 4))
    return _append(None, T, H, H_kv, D, rot, page, dtype, rng.random() < 0.5, rng.random() < 0.5,
                   rng.random() < 0.5, far)


# ------------------------------------------------------------------- lengths that a case stands for
def _share(b):
    """A golden-ratio sequence in (0, 1]: spreads evenly, its first member is the largest."""
    return 1.0 if b == 0 else (b * 0.6180339887498949) % 1.0


def _news(case):
    """Each sequence's (cached slots before, new tokens)."""
    B, n, past = case["B"], case["n"], case["history"]
    if not case["ragged"]:
        return [(past, n)] * B
    return [(int(past * _share(b)), 0 if b % 16 == 9 else max(1, round(n * _share(b + 1 if n < 16 else b))))
            for b in range(B)]


def _members(case):
    """Sequences per group: unequal, none empty."""
    B, P = case["B"], case["groups"]
    weights = [P + 1 - p for p in range(P)]
    out = [1 + (B - P) * w // sum(weights) for w in weights]
    out[0] += B - sum(out)
    return out


def _lengths(case):
    """(length, prefix) of each sequence: its group's shared slots, then 1 to `own` of its own."""
    out = []
    for p, m in enumerate(_members(case)):
        shared = max(1, int(case["prefix"] * _share(p)) // case["page"]) * case["page"]
        out += [(shared + max(1, int(case["own"] * _share(i))), shared) for i in range(m)]
    return out


def _prompts(T):
    """Prompt lengths of a ragged prefill of T tokens: shares of 1/2, 1/3, ... of what is left."""
    out, left, k = [], T, 2
    while left > 0:
        n = max(1, left // k) if len(out) < 7 else left
        out.append(n)
        left -= n
        k = 2 if k == 3 else 3
    return out


# ---------------------------------------------------------------------------------------- the inputs
def _table(g, lengths, page, dev, width=0):
    """Pages in a scattered order for every sequence: (pages in all, page_table)."""
    need = [(n + page - 1) // page for n in lengths]
    total = max(sum(need), 1)
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(lengths), max(max(need), width, 1)), -1, dtype=torch.int32, device=dev)
    used = 0
    for b, m in enumerate(need):
        table[b, :m] = order[used:used + m]
        used += m
    return total, table


def _pages(g, total, H_kv, page, D, dt, dev):
    return tuple(torch.randn(total, H_kv, page, D, generator=g, device=dev, dtype=dt) for _ in "kv")


def _blank(s, lengths, page):
    """Slots past a length hold NaN, as memory that was never written may; the first positions draw
    much attention."""
    first = s["table"][:, 0]
    s["k_pages"][first[first >= 0].unique().long(), :, :min(4, page)] *= 4.0
    for b, n in enumerate(lengths):
        if n % page:
            last = s["table"][b, n // page].long()
            s["k_pages"][last, :, n % page:] = float("nan")
            s["v_pages"][last, :, n % page:] = float("nan")


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    H, H_kv, D = case["H"], case["H_kv"], case["D"]
    s = {"case": case}
    if case["op"] == "prefill":
        news, page = _news(case), case["page"]
        lengths = [past + n for past, n in news]
        total, s["table"] = _table(g, lengths, page, dev)
        s["k_pages"], s["v_pages"] = _pages(g, total, H_kv, page, D, dt, dev)
        _blank(s, lengths, page)
        starts = [0]
        for _, n in news:
            starts.append(starts[-1] + n)
        s["lengths"], s["starts"] = i32(lengths), i32(starts)
        s["q"] = torch.randn(starts[-1], H, D, generator=g, device=dev).to(dt)
    elif case["op"] == "shared":
        page, pairs, first = case["page"], _lengths(case), 0
        lengths = [n for n, _ in pairs]
        # the group's first sequence brings the shared pages, the others pages of their own behind them
        held = []
        for m in _members(case):
            held += [pairs[first][0]] + [n - pre for n, pre in pairs[first + 1:first + m]]
            first += m
        width = max((n + page - 1) // page for n in lengths)
        total, table = _table(g, held, page, dev, width)
        first, groups = 0, [0]
        for m in _members(case):
            k = pairs[first][1] // page
            for b in range(first + 1, first + m):
                table[b] = torch.cat((table[first, :k], table[b, :table.shape[1] - k]))
            first += m
            groups.append(first)
        s["table"] = table
        s["k_pages"], s["v_pages"] = _pages(g, total, H_kv, page, D, dt, dev)
        _blank(s, lengths, page)
        s["lengths"], s["prefix"], s["groups"] = i32(lengths), i32([p for _, p in pairs]), i32(groups)
        s["q"] = torch.randn(case["B"], H, D, generator=g, device=dev).to(dt)
    else:
        T, rot = case["T"], case["rot"]
        # one row of the packed projections per token; q, k and v are slices of it
        s["qkv"] = torch.randn(T, (H + 2 * H_kv) * D, generator=g, device=dev).to(dt)
        # frequencies stretched 8 times over, as for a context 8 times as long
        inv = 500000.0 ** (-torch.arange(0, rot, 2, device=dev).double() / rot)
        s["inv_freq"] = (inv * torch.linspace(1.0, 0.125, rot // 2, device=dev)).float()
        s["factor"] = 1.0 if case.get("in_place") else 0.1 * math.log(8.0) + 1.0
        if case["op"] == "rotary" or not case["prompt"]:
            seq, slot = list(range(T)), [(7 * b + 3) % case.get("page", 16) for b in range(T)]
            lengths = [case.get("page", 16)] * T
            s["positions"] = torch.randint(0, case["far"], (T,), generator=g, device=dev).to(torch.int32)
        else:
            lengths = _prompts(T)
            seq = [b for b, n in enumerate(lengths) for _ in range(n)]
            slot = [i for n in lengths for i in range(n)]
            s["positions"] = i32(slot) + case["far"] // 2
        if case["op"] == "append":
            page = case["page"]
            total, s["table"] = _table(g, lengths, page, dev)
            shape = (total, H_kv, page, D)
            s["k_pages"], s["v_pages"] = (torch.zeros(shape, dtype=dt, device=dev) for _ in "kv")
            s["seq"], s["slots"] = i32(seq), i32(slot)
            s["qw"] = s["kw"] = None
            if case["norm"]:
                s["qw"], s["kw"] = ((1.0 + 0.2 * torch.randn(D, generator=g, device=dev)).to(dt) for _ in "qk")
    return s


# -------------------------------------------------------------------------------- the plain forms
def _slots_of(pages, row, n, page):
    """[H_kv, n, D] in 32 bits: the first n slots of a sequence with the given page-table row."""
    return pages[row[:(n + page - 1) // page].long()].float().transpose(0, 1).flatten(1, 2)[:, :n]


def _softmax_rows(q, k, v, seen):
    """(o, lse) of q [H_kv, rows, D] over k, v [H_kv, n, D]; seen [rows, n] marks a row's slots."""
    score = (q @ k.transpose(1, 2)) * (1.0 / math.sqrt(q.shape[-1]))
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total > 0, total, 1.0)
    return o, (torch.log(total) + top)[..., 0]


def _plain_prefill(s):
    c = s["case"]
    H, H_kv, D, page, window = (c[x] for x in ("H", "H_kv", "D", "page", "window"))
    G, out, lse = H // H_kv, torch.empty_like(s["q"]), s["q"].new_empty(s["q"].shape[:2], dtype=torch.float32)
    at = 0
    for b, (past, n) in enumerate(_news(c)):
        if n == 0:
            continue
        k = _slots_of(s["k_pages"], s["table"][b], past + n, page)
        v = _slots_of(s["v_pages"], s["table"][b], past + n, page)
        slot = torch.arange(past + n, device=k.device)
        for i in range(0, n, 512):
            m = min(512, n - i)
            rows = slice(at + i, at + i + m)
            q = s["q"][rows].float().view(m, H_kv, G, D).transpose(0, 1).reshape(H_kv, m * G, D)
            position = past + i + torch.arange(m, device=k.device).repeat_interleave(G)[:, None]
            seen = slot <= position
            if window:
                seen &= slot > position - window
            o, l = _softmax_rows(q, k, v, seen)
            out[rows] = o.view(H_kv, m, G, D).transpose(0, 1).reshape(m, H, D).to(out.dtype)
            lse[rows] = l.view(H_kv, m, G).transpose(0, 1).reshape(m, H)
        at += n
    return {"o": out, "lse": lse}


def _plain_shared(s):
    c = s["case"]
    H, H_kv, D, page, window = (c[x] for x in ("H", "H_kv", "D", "page", "window"))
    out, lse = torch.empty_like(s["q"]), s["q"].new_empty(s["q"].shape[:2], dtype=torch.float32)
    for b, (n, _) in enumerate(_lengths(c)):
        k = _slots_of(s["k_pages"], s["table"][b], n, page)
        v = _slots_of(s["v_pages"], s["table"][b], n, page)
        slot = torch.arange(n, device=k.device)
        seen = (slot >= (n - window if window else 0))[None]
        o, l = _softmax_rows(s["q"][b].float().view(H_kv, H // H_kv, D), k, v, seen)
        out[b], lse[b] = o.reshape(H, D).to(out.dtype), l.reshape(H)
    return {"o": out, "lse": lse}


def _turned(x, s, c):
    """x [T, heads, D] in 32 bits, rotated: angles in 64 bits, since positions are far."""
    rot = c["rot"]
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    cos, sin = ((s["factor"] * f(angle)).float()[:, None] for f in (torch.cos, torch.sin))
    if c["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _heads(s):
    c = s["case"]
    x = s["qkv"].view(c["T"], c["H"] + 2 * c["H_kv"], c["D"])
    return x[:, :c["H"]], x[:, c["H"]:c["H"] + c["H_kv"]], x[:, c["H"] + c["H_kv"]:]


def _plain_rotary(s):
    c = s["case"]
    q, k, _ = _heads(s)
    new_q, new_k = _turned(q.float(), s, c).to(q.dtype), _turned(k.float(), s, c).to(k.dtype)
    if not c["in_place"]:
        return {"q": new_q, "k": new_k}
    q.copy_(new_q)
    k.copy_(new_k)
    return {"qkv": s["qkv"]}


def _plain_append(s):
    c = s["case"]
    q, k, v = _heads(s)

    def normed(x, w):
        x = x.float()
        return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w.float()

    new_q = _turned(normed(q, s["qw"]), s, c).to(q.dtype)
    new_k = _turned(normed(k, s["kw"]), s, c).to(k.dtype)
    slot = s["slots"].long()
    to = s["table"][s["seq"].long(), slot // c["page"]].long()
    s["k_pages"][to, :, slot % c["page"]] = new_k
    s["v_pages"][to, :, slot % c["page"]] = v
    return {"q": new_q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


PLAIN = {"prefill": _plain_prefill, "shared": _plain_shared, "rotary": _plain_rotary,
         "append": _plain_append}


# ------------------------------------------------------------------------- the framework's operators
_calls = {}


def _framework():
    """The package's operators; its source root is put on the path as its users do."""
    if not _calls:
        import os
        import sys
        sys.path.insert(0, os.path.join(os.getcwd(), "dcr-attention_v3_b200"))
        from dcr_b200.kernel import cuda
        _calls.update(prefill=cuda.paged_prefill, shared=cuda.paged_shared_attention, rotary=cuda.rotary,
                      append=cuda.paged_rotary_append)
    return _calls


def _own(s):
    c = s["case"]
    call = _framework()[c["op"]]
    if c["op"] == "prefill":
        o, lse = call(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["starts"],
                      window=c["window"], return_lse=True)
        return {"o": o, "lse": lse}
    if c["op"] == "shared":
        o, lse = call(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["groups"],
                      s["prefix"], window=c["window"], return_lse=True)
        return {"o": o, "lse": lse}
    q, k, v = _heads(s)
    if c["op"] == "rotary":
        if c["in_place"]:
            call(q, k, s["inv_freq"], s["positions"], interleaved=c["interleaved"], factor=s["factor"],
                 q_out=q, k_out=k)
            return {"qkv": s["qkv"]}
        q, k = call(q, k, s["inv_freq"], s["positions"], interleaved=c["interleaved"], factor=s["factor"])
        return {"q": q, "k": k}
    q = call(q, k, v, s["inv_freq"], s["positions"], s["k_pages"], s["v_pages"], s["table"], s["slots"],
             seq=s["seq"], interleaved=c["interleaved"], factor=s["factor"], q_weight=s["qw"],
             k_weight=s["kw"], eps=1e-5)
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------------------ the work of one pass
def work(case):
    H, H_kv, D, e = case["H"], case["H_kv"], case["D"], BYTES[case["dtype"]]
    if case["op"] == "prefill":
        window, pairs, slots, T = case["window"], 0, 0, 0
        for past, n in _news(case):
            w = window if window else past + n
            # the tokens at positions past .. past + n - 1 see min(position + 1, w) slots each
            full = max(0, min(n, w - past))  # tokens that see all before them
            pairs += full * past + full * (full + 1) // 2 + (n - full) * w
            slots += min(past + n, w + n - 1) if n else 0
            T += n
        return {"bytes": slots * H_kv * D * e * 2 + T * H * (2 * D * e + 4), "flops": 4 * D * H * pairs}
    if case["op"] == "shared":
        window, first, slots, pairs = case["window"], 0, 0, 0
        lengths = _lengths(case)
        for m in _members(case):
            lo = [max(0, n - window) if window else 0 for n, _ in lengths[first:first + m]]
            pre = lengths[first][1]
            slots += max(0, pre - min(lo))
            for (n, p), x in zip(lengths[first:first + m], lo):
                slots += n - max(p, x)
                pairs += n - x
            first += m
        return {"bytes": slots * H_kv * D * e * 2 + case["B"] * H * (2 * D * e + 4),
                "flops": 4 * D * H * pairs}
    T, heads = case["T"], H + H_kv
    flops = 3 * T * heads * case["rot"]
    if case["op"] == "rotary":
        moved = case["rot"] if case["in_place"] else D
        return {"bytes": 2 * T * heads * moved * e + 4 * T + 2 * case["rot"], "flops": flops}
    flops += 4 * T * heads * D if case["norm"] else 0
    return {"bytes": 2 * T * (heads + H_kv) * D * e + 12 * T + 2 * case["rot"], "flops": flops}


# ------------------------------------------------------------- the definitions, evaluated in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"prefill": _exact_prefill, "shared": _exact_shared, "rotary": _exact_rotary,
            "append": _exact_append}[case["op"]](case, s)


def _exact_attention(q, k_pages, v_pages, row, lo, hi, page):
    """(o [m, G, D], lse [m, G]) of q [m, G, D] (64 bits) of one KV head; token i sees slots [lo, hi)."""
    first, last = int(lo.min()), int(hi.max())
    at = torch.arange(first, last, device=q.device)
    k = k_pages[row[at // page].long(), at % page].double()
    v = v_pages[row[at // page].long(), at % page].double()
    hidden = ((at < lo[:, None]) | (at >= hi[:, None]))[:, None]
    z = torch.einsum("mgd,nd->mgn", q, k).div_(math.sqrt(q.shape[-1])).masked_fill_(hidden, -math.inf)
    lse = torch.logsumexp(z, -1)
    return torch.einsum("mgn,nd->mgd", z.sub_(lse[..., None]).exp_(), v), lse


def _exact_prefill(c, s):
    H, H_kv, D, page, window = (c[x] for x in ("H", "H_kv", "D", "page", "window"))
    G, T = H // H_kv, s["q"].shape[0]
    o = torch.zeros(T, H, D, dtype=torch.float64, device=s["q"].device)
    lse = torch.zeros(T, H, dtype=torch.float64, device=o.device)
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    for b, n in enumerate(lengths):
        for i in range(starts[b], starts[b + 1], 256):
            j = min(i + 256, starts[b + 1])
            hi = torch.arange(i, j, device=o.device) + 1 + n - starts[b + 1]
            lo = (hi - window).clamp(min=0) if window else torch.zeros_like(hi)
            for h in range(H_kv):
                heads = slice(h * G, (h + 1) * G)
                o[i:j, heads], lse[i:j, heads] = _exact_attention(
                    s["q"][i:j, heads].double(), s["k_pages"][:, h], s["v_pages"][:, h], s["table"][b],
                    lo, hi, page)
    return {"o": o, "lse": lse}


def _exact_shared(c, s):
    H, H_kv, D, page, window = (c[x] for x in ("H", "H_kv", "D", "page", "window"))
    G = H // H_kv
    o = torch.zeros(c["B"], H, D, dtype=torch.float64, device=s["q"].device)
    lse = torch.zeros(c["B"], H, dtype=torch.float64, device=o.device)
    for b, n in enumerate(s["lengths"].tolist()):
        hi = torch.tensor([n], device=o.device)
        lo = torch.tensor([max(0, n - window) if window else 0], device=o.device)
        for h in range(H_kv):
            heads = slice(h * G, (h + 1) * G)
            o[b, heads], lse[b, heads] = (x[0] for x in _exact_attention(
                s["q"][b:b + 1, heads].double(), s["k_pages"][:, h], s["v_pages"][:, h], s["table"][b],
                lo, hi, page))
    return {"o": o, "lse": lse}


def _exact_turned(x, c, s):
    """Pairs as complex numbers, times factor * exp(i * position * frequency)."""
    rot = c["rot"]
    angle = torch.outer(s["positions"].double(), s["inv_freq"].double())[:, None]
    turn = torch.polar(torch.full_like(angle, s["factor"]), angle)
    x = x.double()
    y = x.clone()
    if c["interleaved"]:
        z = torch.view_as_complex(x[..., :rot].unflatten(-1, (-1, 2)).contiguous()) * turn
        y[..., :rot] = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * turn
        y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
    return y


def _exact_rotary(c, s):
    q, k, v = _heads(s)
    q, k = _exact_turned(q, c, s), _exact_turned(k, c, s)
    if c["in_place"]:
        return {"qkv": torch.cat((q, k, v.double()), 1).flatten(1)}
    return {"q": q, "k": k}


def _exact_append(c, s):
    q, k, v = _heads(s)

    def normed(x, w):
        x = x.double()
        return x if w is None else x / torch.sqrt(x.square().sum(-1, keepdim=True) / c["D"] + 1e-5) * w.double()

    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    seq, slots = s["seq"].long(), s["slots"].long()
    page, at = s["table"][seq, slots // c["page"]].long(), slots % c["page"]
    kp[page, :, at] = _exact_turned(normed(k, s["kw"]), c, s)
    vp[page, :, at] = v.double()
    return {"q": _exact_turned(normed(q, s["qw"]), c, s), "k_pages": kp, "v_pages": vp}
