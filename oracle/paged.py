"""Oracle: the paged key/value cache and attention over it (64 bits, CPU, test infrastructure)."""
from __future__ import annotations

import math

import torch


def kv_quantise(x):
    """(codes as the fp32 values they stand for, scale fp32) of rows x [..., D]: with
    m = max(max|x|, 2**-24), scale = m / 448 and code = e4m3(x * (448 / m)), in fp32 like the
    format's definition; a row that is not finite has scale NaN and codes 0."""
    x = x.float()
    bad = ~torch.isfinite(x).all(-1)
    m = torch.where(bad[..., None], torch.zeros_like(x), x).abs().amax(-1).clamp_min(2.0 ** -24)
    code = torch.where(bad[..., None], torch.zeros_like(x), x * torch.div(torch.full_like(m, 448.0), m)[..., None])
    code = code.clamp(-448, 448).to(torch.float8_e4m3fn).float()
    return code, torch.where(bad, torch.full_like(m, math.nan), m / 448.0)


def kv_values(pool, scale):
    """The rows a pool [pages, kv_heads, page, D] (and its scales) stands for, in 64 bits."""
    x = pool.float().double()
    return x if scale is None else x * scale.double()[..., None]


def paged_attention(q, k, v, page_table, kv_len, cu_q, scale, causal):
    """(o, lse, weight) in 64 bits; k, v are kv_values. Request b: query rows cu_q[b] .. cu_q[b + 1],
    positions j < kv_len[b] on pages page_table[b, j // page]; row i of n sees j <= L - n + i (causal)
    or every j. o = softmax(scale q.k) v (0 for a row that sees nothing), lse natural log [H, T],
    weight = softmax(..) |v|, which bounds what a relative error of the weights does to o. A page
    outside the pool makes the scores of its positions NaN."""
    T, H, D = q.shape
    pages, HKV, page, _ = k.shape
    o = torch.zeros(T, H, D, dtype=torch.float64)
    w = torch.zeros(T, H, D, dtype=torch.float64)
    lse = torch.full((H, T), -math.inf, dtype=torch.float64)
    for b in range(len(kv_len)):
        t0, t1, L = int(cu_q[b]), int(cu_q[b + 1]), max(int(kv_len[b]), 0)
        for t in range(t0, t1):
            stop = min(L, L - (t1 - t0) + (t - t0) + 1) if causal else L
            if stop <= 0:
                continue
            j = torch.arange(stop)
            pg, off = page_table[b].long()[j // page], j % page
            good = (pg >= 0) & (pg < pages)
            for h in range(H):
                kh = k[pg.clamp(0, pages - 1), h // (H // HKV), off]
                vh = v[pg.clamp(0, pages - 1), h // (H // HKV), off]
                s = torch.where(good, (kh @ q[t, h].double()) * scale, math.nan)
                lse[h, t] = torch.logsumexp(s, 0)
                p = torch.softmax(s, 0)
                o[t, h], w[t, h] = p @ vh, p @ vh.abs()
    return o, lse, w
