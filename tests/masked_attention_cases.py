"""Inputs and 64-bit results of the window and tree attention tests (tests/test_gpu_masked_attention.py)."""
import math

import torch


def make(rows, past, hq, hkv, dim, page, dtype, seed, fill=0.0, extra_pages=2, shorter=()):
    """One ragged batch: request r has rows[r] rows behind past[r] keys, in shuffled pages; the caches hold `fill` elsewhere.
    Returns q, k_cache, v_cache, block_table, q_start, kv_len on the host."""
    g = torch.Generator().manual_seed(seed)
    keys = [max(0, p + n) for p, n in zip(past, rows)]
    need = [-(-k // page) for k in keys]
    n_pages = sum(need) + extra_pages
    order = torch.randperm(n_pages - 1, generator=g) + 1
    kc, vc = (torch.full((n_pages, page, hkv, dim), fill, dtype=dtype) for _ in range(2))
    bt = torch.zeros(len(rows), max(1, max(need)), dtype=torch.int32)
    at = 0
    for r, n in enumerate(need):
        pages = order[at:at + n]
        at += n
        bt[r, :n] = pages.to(torch.int32)
        for cache in (kc, vc):
            x = torch.full((n * page, hkv, dim), fill, dtype=dtype)
            x[:keys[r]] = torch.randn(keys[r], hkv, dim, generator=g).to(dtype)
            cache[pages] = x.view(n, page, hkv, dim)
    q = torch.randn(sum(rows), hq, dim, generator=g).to(dtype)
    start = torch.tensor([0] + [sum(rows[:r + 1]) for r in range(len(rows))], dtype=torch.int32)
    return q, kc, vc, bt, start, torch.tensor(keys, dtype=torch.int32)


def sliding_mask(n, L, window, sinks):
    p, j = torch.arange(L - n, L)[:, None], torch.arange(L)[None]
    return (j <= p) & ((j > p - window) | (j < sinks))


def tree_mask(words, n, L):
    """words: int32 [n, words] of one request."""
    mask = torch.zeros(n, L, dtype=torch.bool)
    mask[:, :max(0, L - n)] = True
    for d in range(min(n, 32 * words.shape[1])):
        at = L - n + d
        if at >= 0:
            mask[:, at] = (words[:, d // 32].long() >> d % 32 & 1).bool()
    return mask


def reference(q, kc, vc, bt, start, kv_len, masks, scale=None):
    """(out, weighted) in 64 bits: weighted = sum of the weights times |v|, what the errors of the weights are measured by.
    Masked keys are left out of the sums, so what they hold does not matter."""
    T, hq, dim = q.shape
    page, hkv = kc.shape[1], kc.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    out, weighted = (torch.zeros(T, hq, dim, dtype=torch.float64) for _ in range(2))
    for r in range(len(kv_len)):
        a, b, L = int(start[r]), int(start[r + 1]), int(kv_len[r])
        if a == b:
            continue
        L_there = min(L, bt.shape[1] * page)
        pages = bt[r, :-(-L_there // page)].long()
        mask = masks[r][:, :L_there]
        seen = mask.any(0)
        k, v = (t[pages].reshape(-1, hkv, dim)[:L_there].double() for t in (kc, vc))
        k, v = torch.where(seen[:, None, None], k, 0.0), torch.where(seen[:, None, None], v, 0.0)
        kk, vv = (t.repeat_interleave(hq // hkv, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q[a:b].double(), kk) * scale
        s = s.masked_fill(~mask[None], -math.inf)
        w = torch.nan_to_num(s.softmax(-1), nan=0.0)   # of rows that see nothing
        out[a:b] = torch.einsum("hqk,khd->qhd", w, vv)
        weighted[a:b] = torch.einsum("hqk,khd->qhd", w, vv.abs())
    return out, weighted


def tolerance(out, weighted, dtype, keys):
    """How far an output may be off. half = half a step of the type. The output's rounding: half |out|. A weight is rounded once
    for the product: half of each, so half * weighted. Its exponent is the difference of two 32-bit sums of dim products of
    normal values (below 128 * 2^-24 * 128 * scale = 1.1e-4 for dim 128) and its power of two is good to 2^-13 at worst:
    together below 3e-4 * weighted. fp16 weights below 2^-14 have steps of 2^-24: half of that for each key, times |v| < 6,
    relative to a sum of at least 1."""
    half = torch.finfo(dtype).eps / 2
    small = keys * 2.0 ** -25 * 6 if dtype == torch.float16 else 0.0
    return half * out.abs() + (half + 3e-4) * weighted + small + 1e-30
