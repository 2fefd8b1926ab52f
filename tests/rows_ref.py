"""Definitions of attention over pages for many query rows, of shared prefixes and of rotations in 64
bits, and error bounds that follow from how the kernels compute."""
from __future__ import annotations

import math

import torch

from paged_ref import EPS, UNIT


def attend(q, k_pages, v_pages, rows, lo, hi, *, scale=None, weight_unit=None):
    """(O, lse, bound of O, bound of lse) in float64 of q [T, H, D]: token t sees the slots [lo[t], hi[t])
    of the page-table row rows[t] (int32 [T, max_pages]; -1: not mapped). ``weight_unit``: relative
    rounding of a weight before the second product."""
    T, H, D = q.shape
    H_kv, page = k_pages.shape[1], k_pages.shape[2]
    G, dev = H // H_kv, q.device
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    o = torch.zeros(T, H, D, dtype=torch.float64, device=dev)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64, device=dev)
    tol_o, tol_lse = torch.zeros_like(o), torch.zeros_like(lse)
    lo, hi = (torch.as_tensor(x, device=dev).long() for x in (lo, hi))
    t0 = 0
    while t0 < T:  # a run of tokens with one page-table row
        t1 = t0
        while t1 < T and t1 - t0 < 256 and torch.equal(rows[t1], rows[t0]):
            t1 += 1
        at = torch.arange(int(lo[t0:t1].min()), max(int(hi[t0:t1].max()), 0), device=dev)
        at = at[rows[t0, at // page] >= 0]
        seen = ((at >= lo[t0:t1, None]) & (at < hi[t0:t1, None]))[:, None]
        n = seen.sum(-1).double()
        if len(at):
            pg = rows[t0, at // page].long()
            for h in range(H_kv):
                k = k_pages[pg, h, at % page].double()
                v = v_pages[pg, h, at % page].double()
                heads = slice(h * G, (h + 1) * G)
                x = q[t0:t1, heads].double()
                z = scale * torch.einsum("tgd,nd->tgn", x, k)
                z = torch.where(seen, z, -math.inf)
                s = torch.logsumexp(z, -1)
                p = torch.where(seen, torch.exp(z - torch.where(torch.isinf(s), 0.0, s)[..., None]), 0.0)
                # only the seen slots of a row enter its sums
                blank = torch.where(torch.isfinite(v), v, 0.0)
                o[t0:t1, heads] = torch.einsum("tgn,nd->tgd", p, blank)
                lse[t0:t1, heads] = s
                z0 = torch.where(seen, z, 0.0)
                # the products enter with their absolute sizes, the scale with its own (it may be negative)
                dz = torch.where(seen, abs(scale) * torch.einsum("tgd,nd->tgn", x.abs(), k.abs()), 0.0)
                dz = dz.amax(-1) * (D + 4) * EPS + 4 * EPS * z0.abs().amax(-1)
                rel = 2 * dz + (n + 48) * 2 * EPS
                rel_o = rel + (weight_unit or 0.0)
                part = torch.einsum("tgn,nd->tgd", p, blank.abs())
                u = UNIT[q.dtype]
                tol_o[t0:t1, heads] = u * (o[t0:t1, heads].abs() + rel_o[..., None] * part) + rel_o[..., None] * part
                if q.dtype == torch.float16:  # weights and results below fp16's smallest step are lost
                    tol_o[t0:t1, heads] += n[..., None] * 2.0 ** -25 * blank.abs().amax() + 2.0 ** -25
                tol_lse[t0:t1, heads] = rel + 4 * EPS * torch.where(torch.isinf(s), 0.0, s).abs()
        t0 = t1
    return o, lse, tol_o + 1e-30, tol_lse + 1e-30


def prefill_limits(starts, lengths, window, causal):
    """(lo, hi, sequence) of each token."""
    lo, hi, seq = [], [], []
    for b, n in enumerate(lengths):
        m = starts[b + 1] - starts[b]
        for i in range(m):
            x = n - m + i
            lo.append(max(0, x + 1 - window) if window else 0)
            hi.append(x + 1 if causal else n)
            seq.append(b)
    return lo, hi, seq


def turn(x, positions, inv_freq, interleaved, factor, dt, weight=None, eps=1e-5):
    """(rows, bound) of the rotation of x [T, heads, D] in float64, after a norm where there is a weight."""
    x = x.double()
    rel = 0.0
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
        rel = (x.shape[-1] / 2 + 16) * EPS  # a sum of D squares, rsqrt, products
    r = 2 * len(inv_freq)
    angle = positions.double()[:, None, None] * inv_freq.double()
    z = torch.polar(torch.full_like(angle, factor), angle)
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
    y = torch.complex(a.contiguous(), b.contiguous()) * z
    size = abs(factor) * (a.abs() + b.abs())
    pair = (lambda u, w: torch.stack((u, w), -1).flatten(-2)) if interleaved else (
        lambda u, w: torch.cat((u, w), -1))
    out = torch.cat((pair(y.real, y.imag), x[..., r:]), -1)
    # an angle in half turns rounded to fp32 (2^-25 of one, times pi), its cosine or sine (2 ulp), the
    # factor, two products and a sum
    err = pair(size, size) * (2.0 ** -23 + 2.0 ** -23 + 5 * EPS + 2 * rel)
    err = torch.cat((err, x[..., r:].abs() * rel), -1)
    u = torch.full_like(out, UNIT[dt])
    if weight is None:
        u[..., r:] = 0.0  # copied
    least = 2.0 ** -25 if dt == torch.float16 else 1e-30
    return out, u * (out.abs() + err) + err + least
