"""Definitions of the paged serving operators in 64 bits, slot by slot, and error bounds that
follow from how the kernels compute (fp32 sums, 16-bit weights in two parts, one rounding)."""
from __future__ import annotations

import math

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # ulp/2 of 1
EPS = 2.0 ** -24  # fp32 unit roundoff


def make_pool(lengths, H_kv, page, D, dt, dev, g, *, layout="hnd", extra_pages=2, width=None,
              garbage=float("nan")):
    """Scattered pages: (k_pages, v_pages, page_table). What no sequence holds is ``garbage``."""
    need = [-(-n // page) for n in lengths]
    total = sum(need) + extra_pages
    order = torch.randperm(total, generator=g, device=dev)
    table = torch.full((len(lengths), max(1, width or 0, *need)), -1, dtype=torch.int32, device=dev)
    used = 0
    for b, m in enumerate(need):
        table[b, :m] = order[used:used + m].int()
        used += m
    shape = (total, H_kv, page, D) if layout == "hnd" else (total, page, H_kv, D)
    k = torch.full(shape, garbage, dtype=dt, device=dev)
    v = torch.full(shape, garbage, dtype=dt, device=dev)
    if layout == "nhd":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    for b, n in enumerate(lengths):
        if n:
            at = torch.arange(n, device=dev)
            pg = table[b, at // page].long()
            k[pg, :, at % page] = torch.randn(n, H_kv, D, generator=g, device=dev).to(dt)
            v[pg, :, at % page] = torch.randn(n, H_kv, D, generator=g, device=dev).to(dt)
    return k, v, table


def attend(q, k_pages, v_pages, table, lengths, window=0, scale=None):
    """(O, lse, per-slot weights, bounds of O, lse and weights) in float64."""
    B, H, D = q.shape
    H_kv, page = k_pages.shape[1], k_pages.shape[2]
    G, cap, dev = H // H_kv, table.shape[1] * page, q.device
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    o = torch.zeros(B, H, D, dtype=torch.float64, device=dev)
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device=dev)
    w = torch.zeros(B, H_kv, cap, dtype=torch.float64, device=dev)
    tol_o, tol_lse, tol_w = torch.zeros_like(o), torch.zeros(B, H, dtype=torch.float64, device=dev), torch.zeros_like(w)
    for b, n in enumerate(lengths):
        at = torch.arange(max(0, n - window) if window else 0, n, device=dev)
        at = at[table[b, at // page] >= 0]
        if not len(at):
            continue
        pg = table[b, at // page].long()
        for h in range(H_kv):
            k = k_pages[pg, h, at % page].double()
            v = v_pages[pg, h, at % page].double()
            qs = q[b, h * G:(h + 1) * G].double()
            z = scale * (qs @ k.T)
            p = torch.softmax(z, -1)
            rows = slice(h * G, (h + 1) * G)
            o[b, rows] = p @ v
            lse[b, rows] = torch.logsumexp(z, -1)
            w[b, h, at] = p.sum(0)
            # fp32 dot of D products, its scaling, the exponential of a base-2 score and the
            # subtraction of the maximum; the sums over n slots
            dz = (scale * (qs.abs() @ k.abs().T) * (D + 4)).amax(-1) * EPS + 4 * EPS * z.abs().amax(-1)
            rel = 2 * dz + (len(at) + 32) * 2 * EPS
            u = UNIT[q.dtype]
            if q.dtype != torch.float32:
                rel = rel + 2.0 ** -16  # a weight in two parts of at least 8 bits each
            part = p @ v.abs()
            tol_o[b, rows] = u * (o[b, rows].abs() + rel[:, None] * part) + rel[:, None] * part
            if q.dtype == torch.float16:  # parts below fp16's smallest step are lost
                tol_o[b, rows] += len(at) * 2.0 ** -25 * v.abs().amax()
            tol_lse[b, rows] = rel + 4 * EPS * lse[b, rows].abs()
            slot_rel = 4 * dz + (len(at) + 64) * 2 * EPS + 4 * EPS * lse[b, rows].abs()
            tol_w[b, h, at] = (p * slot_rel[:, None]).sum(0)
    tol_o += 1e-30
    return o, lse, w, tol_o, tol_lse + 1e-30, tol_w + 1e-30


def norm_rotate(x, weight, cos, sin, eps, dt):
    """(rows, bound) of norm and rotation of x [T, heads, D] with cos, sin [T, D] in float64."""
    x = x.double()
    D = x.shape[-1]
    if weight is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + eps) * weight.double()
    a, b = x[..., :D // 2], x[..., D // 2:]
    c, s = cos.double()[:, None], sin.double()[:, None]
    y = torch.cat((a * c[..., :D // 2] - b * s[..., :D // 2],
                   b * c[..., D // 2:] + a * s[..., D // 2:]), -1)
    size = torch.cat(((a * c[..., :D // 2]).abs() + (b * s[..., :D // 2]).abs(),
                      (b * c[..., D // 2:]).abs() + (a * s[..., D // 2:]).abs()), -1)
    # half the relative error of a sum of D squares, rsqrt (2 ulp), four products, a sum
    rel = (D / 2 + 16) * EPS
    # fp16 values below 2^-14 are subnormal: steps of 2^-24, so a rounding error of 2^-25
    least = 2.0 ** -25 if dt == torch.float16 else 1e-30
    return y, UNIT[dt] * (y.abs() + rel * size) + rel * size + least


def evict(weights, pos, n, seen, budget, sinks, recent):
    """src of one row (python lists), the definition: sort by claim, fill holes in slot order."""
    nan = [w != w for w in weights]
    sure = [p < sinks or p >= seen - recent for p in pos]

    def claim(i):
        if sure[i]:
            return (0, 0.0, i)
        return (1, 0.0, i) if nan[i] else (2, -weights[i], i)
    kept = set(sorted(range(n), key=claim)[:budget])
    late = iter([i for i in range(budget, n) if i in kept])
    m = min(n, budget)
    return [i if i in kept else next(late) for i in range(m)] + [-1] * (budget - m)


def logits(x, tokens, n, prompt, rep, pres, freq, bias, allowed):
    """(row, bound, allowed mask) of one row in float64."""
    V = x.shape[0]
    dt = x.dtype
    x = x.double()
    t = torch.as_tensor(tokens[:n], device=x.device).long()
    m = torch.as_tensor(tokens[prompt:n] if prompt < n else [], device=x.device).long()
    every = torch.bincount(t[t >= 0], minlength=V)[:V]
    said = torch.bincount(m[m >= 0], minlength=V)[:V].double()
    y = torch.where(every > 0, torch.where(x > 0, x / rep, x * rep), x)
    size = y.abs() + said * abs(freq) + abs(pres)
    y = y - said * freq - (said > 0) * pres
    if bias is not None:
        y = y + bias.double()
        size = size + bias.double().abs()
    ok = torch.ones(V, dtype=torch.bool, device=x.device)
    if allowed is not None:
        i = torch.arange(V, device=x.device)
        ok = ((allowed.long()[i // 32] >> (i % 32)) & 1) == 1
        y = torch.where(ok, y, -math.inf)
    tol = UNIT[dt] * size * (1 + 2 * UNIT[dt]) + 6 * EPS * size + 1e-30
    if dt == torch.float16:
        tol = tol + 2.0 ** -25  # subnormal steps
    return y, tol, ok
