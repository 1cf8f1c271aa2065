"""Plain 64-bit forms of the rotation, the paged append and paged attention, and
how far the kernels may be from them.

A bf16 rounding is off by at most 2^-8 of the value (half a step), one in fp32 by
2^-24."""
from __future__ import annotations

import math

import torch

BF = torch.bfloat16


def rotate(x, positions, turns, interleaved=False, magnitude=1.0, inverse=False):
    """x [tokens, heads, D] in 64 bits; positions [tokens]."""
    n = turns.numel()
    angle = torch.remainder(positions.double()[:, None] * turns.double(), 1.0)[:, None] * (2 * math.pi)
    c, s = torch.cos(angle) * magnitude, torch.sin(angle) * magnitude * (-1.0 if inverse else 1.0)
    y = x.clone()
    ia = torch.arange(0, 2 * n, 2, device=x.device) if interleaved else torch.arange(n, device=x.device)
    ib = ia + 1 if interleaved else ia + n
    a, b = x[..., ia], x[..., ib]
    y[..., ia] = a * c - b * s
    y[..., ib] = b * c + a * s
    return y


def rotate_bound(x, want, turns, interleaved=False, magnitude=1.0):
    """2^-8 of the result, and 2^-20 m (|a| + |b|) for fp32: the angle is off by
    pi 2^-24 and its sine and cosine by 2^-22 (two ulps), the products and their
    sum by 4 x 2^-24, together below 2^-20.7.  Passed dims are copies."""
    n = turns.numel()
    ia = torch.arange(0, 2 * n, 2, device=x.device) if interleaved else torch.arange(n, device=x.device)
    ib = ia + 1 if interleaved else ia + n
    bound = torch.zeros_like(want)
    both = (x[..., ia].abs() + x[..., ib].abs()) * abs(magnitude) * 2.0**-20
    bound[..., ia] = want[..., ia].abs() * 2.0**-8 + both * 1.01
    bound[..., ib] = want[..., ib].abs() * 2.0**-8 + both * 1.01
    return bound


def places(q_start, kv_len, page_table, page_size, tokens):
    """Per token (sequence, position); sequences' tokens only."""
    out = []
    qs = q_start.tolist() if q_start is not None else list(range(len(kv_len) + 1))
    for b, kv in enumerate(kv_len.tolist()):
        kv = min(max(kv, 0), page_table.shape[1] * page_size)
        n = qs[b + 1] - qs[b]
        out += [(qs[b] + i, b, kv - n + i) for i in range(n)]
    return out


def attend(q, k_cache, v_cache, page_table, q_start, kv_len, scale, causal=True, window=0):
    """(o, bound) [tokens, heads, D] in 64 bits; rows of no sequence are NaN.

    A key takes part with its own row or not at all, so what hidden rows hold does
    not show.  With w the weights: the scores are off by e = (D + 4) 2^-24 |scale|
    sum |q k| each (fp32 sum, products by scale log2 e, the running maximum), the
    exponential by 2^-22, the weight by 2^-8 where it is rounded to bf16 for the
    matrix unit; the two sums of n terms by n 2^-24 each.  The output moves by at
    most the sum of these times (sum w |v| / sum w + |o|), and 2^-8 |o| at the end."""
    T, Hq, D = q.shape
    pages, Hkv, P, _ = k_cache.shape
    G = Hq // Hkv
    o = torch.full((T, Hq, D), float("nan"), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(o)
    qs = q_start.tolist() if q_start is not None else list(range(kv_len.numel() + 1))
    for b, kv in enumerate(kv_len.tolist()):
        kv = min(max(kv, 0), page_table.shape[1] * P)
        q0, n = qs[b], qs[b + 1] - qs[b]
        if n == 0:
            continue
        j = torch.arange(kv, device=q.device)
        page = page_table[b][j // P].long() if kv else j
        there = (page >= 0) & (page < pages)
        page = torch.where(there, page, 0)
        K = k_cache[page, :, j % P].double()  # [kv, Hkv, D]
        V = v_cache[page, :, j % P].double()
        limit = kv - n + torch.arange(n, device=q.device)
        seen = there[None, :].expand(n, kv)
        if causal:
            seen = seen & (j[None, :] <= limit[:, None])
        if window:
            seen = seen & (j[None, :] > limit[:, None] - window)
        for h in range(Hq):
            x = q[q0:q0 + n, h].double()
            k, v = K[:, h // G], V[:, h // G]
            any_seen = seen.any(0)
            k = torch.where(any_seen[:, None], k, 0.0)
            s = (x @ k.T.contiguous()) * scale
            mag = (x.abs() @ k.abs().T.contiguous()) * abs(scale)
            s = torch.where(seen, s, float("-inf"))
            top = s.amax(-1, keepdim=True) if kv else torch.zeros(n, 1, dtype=torch.float64, device=q.device)
            w = torch.where(seen, torch.exp(s - torch.where(torch.isinf(top) & (top < 0), 0.0, top)), 0.0)
            L = w.sum(-1, keepdim=True)
            bad = ~torch.isfinite(v)
            fine = torch.where(bad, 0.0, v)
            num = w @ fine
            if bool(bad.any()):  # rows that see a value that is no number: its products, others none
                for r in range(n):
                    vis = seen[r] & bad.any(-1)
                    if bool(vis.any()):
                        num[r] = (w[r][seen[r]][:, None] * v[seen[r]]).sum(0)
            A = torch.where(L > 0, (w @ fine.abs()) / L, 0.0)
            r = torch.where(L > 0, num / L, torch.where(torch.isnan(L), L, 0.0))
            e = (D + 4) * 2.0**-24 * torch.where(seen, mag, 0.0).amax(-1, keepdim=True) if kv else torch.zeros_like(L)
            eps = 2.0**-8 + 2.0**-22 + 2 * e + 2 * kv * 2.0**-24
            o[q0:q0 + n, h] = r
            bound[q0:q0 + n, h] = 1.01 * (2.0**-8 * r.abs() + eps * (A + r.abs())) + 2.0**-133
    return o, bound


def far(got, want, bound):
    """Values outside the bound, or finite where they should not be."""
    got = got.double()
    ok = torch.where(torch.isfinite(want), (got - want).abs() <= bound,
                     torch.where(torch.isnan(want), torch.isnan(got), got == want))
    return int((~ok).sum())
