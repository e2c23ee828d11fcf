"""The paged operators in float64 on the CPU, written from their definitions, and the error bounds the GPU tests use."""
import math

import torch

F64 = torch.float64
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # torch.finfo(t).eps / 2


def keys_of(pool, pages, n):
    """The first n rows of a list of pages of a pool [n_pages, kv_heads, page_size, hd]: [kv_heads, n, hd]."""
    ps = pool.shape[2]
    rows = [pool[int(pages[j // ps]), :, j % ps] for j in range(n)]
    return torch.stack(rows, 1).to(F64) if rows else torch.zeros(pool.shape[1], 0, pool.shape[3], dtype=F64)


def attention(q, k, v, table, kv_lens, cu_q, heads, scale, cap=0.0, slopes=None, prefix_lens=None, causal=True, prefix=None):
    """q [tokens, heads * hd] and the pools on the CPU -> (out, lse, bound of |out - exact|, bound of |lse - exact|), all
    float64; rows behind the last sequence are NaN.  prefix: (page numbers, keys) of a prefix that every token sees.

    The bound.  With u = half a step of the type: the result is rounded once (u |out|) and each softmax weight once
    before the second product (u sum p |v|, for f16 also n 2^-25 max |v|, what a weight below its smallest step can
    lose against a largest weight of 1).  A score's error e (below) changes its weight, and the sum, by e relatively: 2 e sum
    p |v|.  32-bit sums over n keys in any order add at most 2 (n / 16 + 64) 2^-24 sum p |v| (the tensor core adds 16 at
    a time), exp2 and the divisions 2^-20.
    e = (hd + 8) 2^-24 |scale| sum |q| |k| (the dot product; a bound has no sign) + 16 2^-24 cap (tanh by one exponential and one reciprocal) +
    4 2^-24 |bias| + 2^-21 max |score| (products with scale and log2 e)."""
    tokens, kvh, hd = q.shape[0], k.shape[1], k.shape[3]
    group, u = heads // kvh, HALF_STEP[k.dtype]
    out = torch.full((tokens, heads, hd), float("nan"), dtype=F64)
    lse = torch.full((tokens, heads), float("nan"), dtype=F64)
    tol, ltol = out.clone(), lse.clone()
    q = q.to(F64).reshape(tokens, heads, hd)
    off = prefix[1] if prefix else 0
    pre = [keys_of(p, prefix[0], off) for p in (k, v)] if prefix else None
    for b, n in enumerate(kv_lens):
        lo, hi = (b, b + 1) if cu_q is None else (cu_q[b], cu_q[b + 1])
        kk, vv = keys_of(k, table[b], n), keys_of(v, table[b], n)
        if prefix:
            kk, vv = torch.cat([pre[0], kk], 1), torch.cat([pre[1], vv], 1)
        for t in range(lo, hi):
            place = n - (hi - lo) + (t - lo)
            see = n if not causal else min(n, max(place + 1, 0, prefix_lens[b] if prefix_lens is not None else 0))
            see += off
            for h in range(heads):
                if see == 0:
                    out[t, h], lse[t, h], tol[t, h], ltol[t, h] = 0.0, -math.inf, 0.0, 0.0
                    continue
                K, V = kk[h // group, :see], vv[h // group, :see]
                s = K @ q[t, h] * scale
                e = (hd + 8) * 2.0 ** -24 * abs(scale) * (K.abs() @ q[t, h].abs()).max()
                if cap:
                    s = cap * torch.tanh(s / cap)
                    e += 16 * 2.0 ** -24 * cap
                if slopes is not None:
                    bias = float(slopes[h]) * (off + place - torch.arange(see, dtype=F64)).abs()
                    s = s - bias
                    e += 4 * 2.0 ** -24 * bias.max()
                e = float(e + 2.0 ** -21 * s.abs().max())
                m = s.max()
                p = torch.exp(s - m)
                lse[t, h] = m + torch.log(p.sum())
                p = p / p.sum()
                out[t, h] = p @ V
                A = p @ V.abs()
                tol[t, h] = u * out[t, h].abs() + (u + 2 * e + 2 * (see / 16 + 64) * 2.0 ** -24 + 2.0 ** -20) * (1 + u) * A
                if k.dtype == torch.float16:
                    tol[t, h] += see * 2.0 ** -25 * V.abs().max() + 2.0 ** -25
                ltol[t, h] = e + (see / 16 + 64) * 2.0 ** -24 + 2.0 ** -20 * (1 + abs(float(lse[t, h])))
    return out.reshape(tokens, -1), lse, tol.reshape(tokens, -1), ltol


def rotate(x, cos, sin):
    """x [tokens, heads, hd] float64 by cos / sin [tokens, r / 2]: (result, bound of the error before rounding)."""
    half = cos.shape[1]
    c, s = cos.to(F64)[:, None], sin.to(F64)[:, None]
    a, b, rest = x[..., :half], x[..., half: 2 * half], x[..., 2 * half:]
    y = torch.cat([a * c - b * s, b * c + a * s, rest], -1)
    mag = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), torch.zeros_like(rest)], -1)
    return y, 2 * 2.0 ** -24 * mag  # two products and a sum in 32 bits


def make(seed, q_lens, kv_lens, heads, kv_heads, hd, ps, dtype, garbage=float("nan"), prefix=0, spare=2, tail=0, width=0):
    """Pools, table and queries on the CPU; pages in a random order, `garbage` wherever no sequence has a key; `tail` rows
    of q belong to nobody; the table has at least `width` columns."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // ps) for n in kv_lens]
    n_pre = -(-prefix // ps)
    n_pages = sum(need) + n_pre + spare
    k = torch.randn(n_pages, kv_heads, ps, hd, generator=g).to(dtype)
    v = torch.randn(n_pages, kv_heads, ps, hd, generator=g).to(dtype)
    perm = torch.randperm(n_pages, generator=g).to(torch.int32)
    table = torch.full((len(kv_lens), max(width, max(need) + 1)), -7, dtype=torch.int32)
    used = torch.zeros(n_pages, ps, dtype=torch.bool)
    at = 0
    for b, n in enumerate(kv_lens):
        table[b, : need[b]] = perm[at: at + need[b]]
        for j in range(n):
            used[int(table[b, j // ps]), j % ps] = True
        at += need[b]
    pre = perm[at: at + n_pre].clone()
    for j in range(prefix):
        used[int(pre[j // ps]), j % ps] = True
    for pool in (k, v):
        pool.transpose(1, 2)[~used] = garbage
    cu = [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1] + tail, heads * hd, generator=g).to(dtype)
    return dict(q=q, k=k, v=v, table=table, cu=cu, pre=pre)
