"""The paged-cache operators as a serving program calls them: what is measured, in plain form and through the framework.

Three operators of ``quanta_b200.paged``:
  append  paged_rope_append: new keys and values into the pages of their sequences, rotated on the way, and rotated queries
  attend  paged_attention: every new token against its sequence's pages (single tokens, prompts, chunks of prompts)
  shared  shared_prefix_attention: the same where the whole batch shares one long prefix, kept once

A case's lengths come from the numbers in the case alone (``_lengths``), the values of its tensors from the seed.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _case(op, name=None, **kw):
    c = {"op": op, "dtype": "bf16", "src": "bf16", "heads": 32, "kv_heads": 8, "hd": 128, "page": 16, "batch": 1, "q_min": 1, "q_max": 1,
         "kv_min": 1, "kv_max": 1, "lens": 1, "rot": 0, "offset": 0, "cap": 0.0, "slopes": False, "prefix_mask": 0, "prefix": 0, "singles": 0.0}
    c.update(kw)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # one decode step of the framework's decoder stack: 16 sequences, 32 heads, f32 projections into a bf16 cache (latency)
        _case("append", "append_tokens_16", src="f32", kv_heads=32, batch=16, kv_min=1024, kv_max=1025, lens=11),
        # five prompts arrive together, about 8000 tokens, shared K/V heads, projections in bf16
        _case("append", "append_prompts", page=64, batch=5, q_min=900, q_max=2400, lens=16),
        # a chunk behind a prefix kept elsewhere: positions shifted, half of the head rotated, fp16
        _case("append", "append_partial_f16", dtype="f16", src="f16", heads=24, kv_heads=6, hd=64, page=32, batch=3, q_min=200, q_max=330, kv_min=400,
              kv_max=900, lens=13, rot=32, offset=5000),
        # one user, one token, a short context: latency alone
        _case("attend", "attend_token_1", kv_min=1024, kv_max=1024, lens=21),
        # the framework's decode step: 16 sequences at context 1024, as many K/V heads as Q heads
        _case("attend", "attend_tokens_16", kv_heads=32, batch=16, kv_min=1024, kv_max=1025, lens=22),
        # a serving batch: 64 sequences between one token and 8192, shared K/V heads
        _case("attend", "attend_tokens_ragged", batch=64, kv_min=1, kv_max=8192, lens=23),
        # one user with a very long context
        _case("attend", "attend_token_long", heads=64, page=64, kv_min=131072, kv_max=131072, lens=24),
        # one prompt of 8192 tokens
        _case("attend", "attend_prompt_8192", page=64, q_min=8192, q_max=8192, lens=25),
        # several prompts of odd lengths, heads of 64, capped scores, fp16
        _case("attend", "attend_prompts_cap_f16", dtype="f16", heads=24, kv_heads=24, hd=64, page=32, batch=5, q_min=301, q_max=2100, lens=26, cap=30.0),
        # a mixed step: chunks of prompts and single tokens in one call, bias by distance, a bidirectional prefix
        _case("attend", "attend_mixed_bias", batch=40, q_min=100, q_max=700, kv_min=100, kv_max=6000, lens=27, slopes=True, prefix_mask=200,
              singles=0.7),
        # 64 sequences behind one system prompt of 8192 tokens, each with its own short tail
        _case("shared", "shared_tokens_64", batch=64, kv_min=1, kv_max=512, lens=31, prefix=8192),
        # a few drafts of three tokens each behind a prefix of odd length, fp16, heads of 64
        _case("shared", "shared_drafts_f16", dtype="f16", heads=12, kv_heads=4, hd=64, page=32, batch=7, q_min=3, q_max=3, kv_min=3, kv_max=90, lens=32,
              prefix=1001),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ones' ranges, its cost bounded by the largest listed ones'."""
    op = rng.choice(["append", "attend", "attend", "attend", "shared"])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 8, 16, 32])
    group = rng.choice([1, 1, 2, 3, 4, 4, 6, 8, 12, 16])
    while kv_heads * group > 64:
        group = max(1, group // 2)
    c = _case(op, dtype=rng.choice(["bf16", "bf16", "f16"]), heads=kv_heads * group, kv_heads=kv_heads, hd=rng.choice([64, 128, 128]),
              page=rng.choice([16, 16, 32, 64, 128]), lens=rng.randrange(1 << 20))
    c["src"] = c["dtype"]
    if op == "append":
        c["src"] = rng.choice(["f32", c["dtype"]])
        c["rot"] = rng.choice([0, 0, c["hd"] // 2])
        c["offset"] = rng.choice([0, 0, rng.randrange(1, 20000)])
        tokens = _log_int(rng, 1, 8192)
        c["batch"] = min(tokens, _log_int(rng, 1, 64))
        c["q_max"] = max(1, tokens // c["batch"])
        c["q_min"] = rng.randrange(1, c["q_max"] + 1)
        c["kv_min"] = rng.randrange(1, 500)
        c["kv_max"] = c["kv_min"] + rng.randrange(0, 2000)
        return c
    c["cap"] = rng.choice([0.0, 0.0, 0.0, 20.0, 50.0])
    c["slopes"] = rng.random() < 0.2
    if op == "shared":
        c["prefix"] = _log_int(rng, 64, 16384)
        c["batch"] = _log_int(rng, 2, 128)
        c["q_max"] = c["q_min"] = rng.choice([1, 1, 1, 2, 5])
        c["kv_min"] = rng.randrange(1, 100)
        c["kv_max"] = c["kv_min"] + rng.randrange(0, 700)
        return c
    if rng.random() < 0.5:  # single tokens, up to about 1 GB of keys and values
        room = (1 << 30) // (4 * c["kv_heads"] * c["hd"])
        c["kv_max"] = _log_int(rng, 1, min(131072, room))
        c["kv_min"] = rng.choice([1, c["kv_max"]])
        c["batch"] = _log_int(rng, 1, max(1, min(128, room // c["kv_max"])))
        return c
    c["q_max"] = _log_int(rng, 1, 4096)  # prompts and chunks of prompts
    c["q_min"] = rng.choice([1, max(1, c["q_max"] // 2), c["q_max"]])
    extra = rng.choice([0, 0, _log_int(rng, 1, 4096)])
    c["kv_min"], c["kv_max"] = rng.choice([1, max(1, extra)]), max(1, c["q_max"] + extra)
    c["prefix_mask"] = rng.choice([0, 0, 0, rng.randrange(1, 600)])
    c["singles"] = rng.choice([0.0, 0.0, 0.6])
    pairs = 8192 * 8192 * 32 * 128 // (2 * 2 * c["heads"] * c["hd"])  # half of the longest listed prompt's products
    c["batch"] = _log_int(rng, 1, max(1, min(32, pairs // (c["q_max"] * c["kv_max"]))))
    return c


def _lengths(c):
    """New tokens and keys (new ones included) of every sequence."""
    r = random.Random(c["lens"])
    q = [r.randint(c["q_min"], c["q_max"]) if c["q_min"] < c["q_max"] else c["q_max"] for _ in range(c["batch"])]
    if c["singles"]:
        q = [1 if r.random() < c["singles"] else n for n in q]
    kv = [max(a, r.randint(c["kv_min"], c["kv_max"])) for a in q]
    return q, kv


def _scale(c):
    return 1.0 / math.sqrt(c["hd"])


def _slopes(c):
    return [2.0 ** (-8.0 * (h + 1) / c["heads"]) for h in range(c["heads"])]


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    q_lens, kv_lens = _lengths(c)
    dt, hd, ps, kvh = TYPES[c["dtype"]], c["hd"], c["page"], c["kv_heads"]
    n_seq = [-(-n // ps) for n in kv_lens]
    n_pre = -(-c["prefix"] // ps)
    need = sum(n_seq) + n_pre
    n_pages = need + max(2, need // 16)  # some pages belong to nobody
    perm = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)
    k = torch.empty(n_pages, kvh, ps, hd, dtype=dt, device=DEV)
    v = torch.empty_like(k)
    k.normal_(generator=gen)
    v.normal_(generator=gen)
    width = max(n_seq) + 1
    table = torch.full((c["batch"], width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(n_seq):
        table[b, :n] = perm[at: at + n]
        at += n
    total = sum(q_lens)
    cu = [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    s = {"case": c, "q_lens": q_lens, "kv_lens": kv_lens, "k": k, "v": v, "table": table, "tokens": total,
         "kv_dev": torch.tensor(kv_lens, dtype=torch.int32, device=DEV),
         "cu_dev": None if max(q_lens) == 1 else torch.tensor(cu, dtype=torch.int32, device=DEV)}
    src = TYPES[c["src"]] if c["op"] == "append" else dt
    # a fused projection's output: q, k and v of a token side by side (append); the attention's own queries are dense
    if c["op"] == "append":
        width = (c["heads"] + 2 * kvh) * hd
        qkv = torch.randn(total, width, generator=gen, device=DEV).to(src)
        a, b2 = c["heads"] * hd, (c["heads"] + kvh) * hd
        s["qn"], s["kn"], s["vn"] = qkv[:, :a], qkv[:, a:b2], qkv[:, b2:]
        rot = c["rot"] or hd
        n_pos = max(kv_lens) + c["offset"]
        ang = torch.arange(n_pos, dtype=torch.float64, device=DEV)[:, None] * torch.pow(
            torch.tensor(10000.0, dtype=torch.float64, device=DEV), -2.0 * torch.arange(rot // 2, dtype=torch.float64, device=DEV) / rot)[None]
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        slots = torch.cat([torch.arange(n - m, n) for m, n in zip(q_lens, kv_lens)])
        seq = torch.cat([torch.full((m,), i, dtype=torch.int64) for i, m in enumerate(q_lens)])
        s["slots"], s["seq"] = slots.to(DEV), seq.to(DEV)
        s["positions"] = (slots + c["offset"]).to(torch.int32).to(DEV) if c["offset"] else None
    else:
        s["q"] = torch.randn(total, c["heads"] * hd, generator=gen, device=DEV).to(dt)
        s["slopes"] = torch.tensor(_slopes(c), dtype=torch.float32, device=DEV) if c["slopes"] else None
        s["prefix_mask"] = torch.full((c["batch"],), c["prefix_mask"], dtype=torch.int32, device=DEV) if c["prefix_mask"] else None
        s["prefix_pages"] = perm[at: at + n_pre].contiguous() if c["prefix"] else None
        # what lies behind the last key of a sequence, and in pages of nobody, is whatever an earlier use left
        nan = float("nan")
        for b, n in enumerate(kv_lens):
            if n % ps:
                p = int(table[b, n // ps]) if c["batch"] <= 64 else None
                if p is not None:
                    k[p, :, n % ps:], v[p, :, n % ps:] = nan, nan
        free = perm[need:].long()
        k[free], v[free] = nan, nan
    if own:
        from quanta_b200 import paged
        s["cache"] = paged.PagedKVCache.from_parts(k, v)
        s["batch"] = paged.PagedBatch(s["cache"], table, s["kv_dev"], s["cu_dev"])
    return s


# ---- the framework's calls ---------------------------------------------------------------------------------------

def _run_own(s):
    from quanta_b200 import paged
    c = s["case"]
    if c["op"] == "append":
        q = paged.paged_rope_append(s["batch"], s["qn"], s["kn"], s["vn"], s["cos"], s["sin"], positions=s["positions"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    if c["op"] == "shared":
        return paged.shared_prefix_attention(s["batch"], s["q"], s["prefix_pages"], c["prefix"], scale=_scale(c), softcap=c["cap"], slopes=s["slopes"])
    return paged.paged_attention(s["batch"], s["q"], scale=_scale(c), softcap=c["cap"], slopes=s["slopes"], prefix_lens=s["prefix_mask"])


# ---- the plain form ----------------------------------------------------------------------------------------------

def _rotate(x, cos, sin):
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half: 2 * half], x[..., 2 * half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], dim=-1)


def _append_plain(s):
    c = s["case"]
    dt, hd, ps = TYPES[c["dtype"]], c["hd"], c["page"]
    pos = s["slots"] if s["positions"] is None else s["positions"].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    q = _rotate(s["qn"].float().reshape(-1, c["heads"], hd), cos, sin).to(dt)
    k = _rotate(s["kn"].float().reshape(-1, c["kv_heads"], hd), cos, sin).to(dt)
    page = s["table"][s["seq"], s["slots"] // ps].long()
    s["k"][page, :, s["slots"] % ps] = k
    s["v"][page, :, s["slots"] % ps] = s["vn"].reshape(-1, c["kv_heads"], hd).to(dt)
    return {"q": q.reshape(-1, c["heads"] * hd), "k": s["k"], "v": s["v"]}


def _keys(s, pages, n):
    """The first n keys and values of a list of pages: [kv_heads, n, hd] in 32 bits."""
    out = []
    for pool in (s["k"], s["v"]):
        x = pool[pages.long()].float()
        out.append(x.permute(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[3])[:, :n])
    return out


def _attend_plain(s):
    c = s["case"]
    dt, hd, ps, kvh = TYPES[c["dtype"]], c["hd"], c["page"], c["kv_heads"]
    group = c["heads"] // kvh
    out = torch.empty(s["tokens"], c["heads"] * hd, dtype=dt, device=DEV)
    pre = c["prefix"]
    shared = _keys(s, s["prefix_pages"], pre) if pre else None
    t0 = 0
    for b, (m, n) in enumerate(zip(s["q_lens"], s["kv_lens"])):
        k, v = _keys(s, s["table"][b, : -(-n // ps)], n)
        if pre:
            k, v = torch.cat([shared[0], k], dim=1), torch.cat([shared[1], v], dim=1)
        total = pre + n
        j = torch.arange(total, device=DEV)
        step = max(1, (1 << 28) // (c["heads"] * total))
        for i0 in range(0, m, step):
            i1 = min(m, i0 + step)
            q = s["q"][t0 + i0: t0 + i1].float().reshape(i1 - i0, kvh, group, hd).permute(1, 0, 2, 3).reshape(kvh, -1, hd)
            sc = torch.matmul(q, k.transpose(1, 2)).reshape(kvh, i1 - i0, group, total) * _scale(c)
            if c["cap"]:
                sc = torch.tanh(sc / c["cap"]) * c["cap"]
            pos = torch.arange(pre + n - m + i0, pre + n - m + i1, device=DEV)
            if s["slopes"] is not None:
                dist = (pos[:, None] - j[None]).abs().float()
                sc = sc - s["slopes"].reshape(kvh, 1, group, 1) * dist[None, :, None, :]
            seen = j[None] < torch.clamp(pos + 1, min=pre + c["prefix_mask"])[:, None]
            sc = torch.where(seen[None, :, None], sc, float("-inf"))
            sc = torch.exp(sc - sc.amax(dim=-1, keepdim=True))
            p = sc / sc.sum(dim=-1, keepdim=True)
            o = torch.matmul(p.reshape(kvh, -1, total), v).reshape(kvh, i1 - i0, group, hd).permute(1, 0, 2, 3)
            out[t0 + i0: t0 + i1] = o.reshape(i1 - i0, -1).to(dt)
        t0 += m
    return out


def run(state):
    if own:
        return _run_own(state)
    return _append_plain(state) if state["case"]["op"] == "append" else _attend_plain(state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def work(case):
    c = case
    q_lens, kv_lens = _lengths(c)
    total, hd, kvh, heads = sum(q_lens), c["hd"], c["kv_heads"], c["heads"]
    if c["op"] == "append":
        src = 4 if c["src"] == "f32" else 2
        rot = c["rot"] or hd
        width = (heads + 2 * kvh) * hd
        return {"bytes": total * (width * (src + 2) + rot * 4), "flops": total * (heads + kvh) * rot * 3}
    keys = sum(kv_lens) + c["prefix"]
    pairs = 0
    for m, n in zip(q_lens, kv_lens):
        for p in range(n - m, n):
            pairs += c["prefix"] + max(p + 1, min(n, c["prefix_mask"]))
    return {"bytes": 2 * (2 * total * heads * hd + 2 * keys * kvh * hd), "flops": 4 * pairs * heads * hd}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------

def exact(case, seed):
    c = case
    s = prepare(case, seed)
    hd, ps, kvh, heads = c["hd"], c["page"], c["kv_heads"], c["heads"]
    group = heads // kvh
    table, f64 = s["table"].long(), torch.float64
    if c["op"] == "append":
        q_new, k_new = s["qn"].to(f64).reshape(-1, heads, hd).clone(), s["kn"].to(f64).reshape(-1, kvh, hd).clone()
        half = s["cos"].shape[1]
        kp, vp = s["k"].to(f64), s["v"].to(f64)
        t = 0
        for b, (m, n) in enumerate(zip(s["q_lens"], s["kv_lens"])):
            slot = torch.arange(n - m, n, device=DEV)
            ca, sa = s["cos"][slot + c["offset"]].to(f64)[:, None], s["sin"][slot + c["offset"]].to(f64)[:, None]
            for x in (q_new, k_new):
                lo, hi = x[t: t + m, :, :half].clone(), x[t: t + m, :, half: 2 * half].clone()
                x[t: t + m, :, :half] = lo * ca - hi * sa
                x[t: t + m, :, half: 2 * half] = hi * ca + lo * sa
            page = table[b][slot // ps]
            kp[page, :, slot % ps] = k_new[t: t + m]
            vp[page, :, slot % ps] = s["vn"][t: t + m].to(f64).reshape(m, kvh, hd)
            t += m
        return {"q": q_new.reshape(-1, heads * hd), "k": kp, "v": vp}
    out = torch.zeros(s["tokens"], heads, hd, dtype=f64, device=DEV)
    slopes = _slopes(c)
    t = 0
    for b, (m, n) in enumerate(zip(s["q_lens"], s["kv_lens"])):
        where = [(int(p), i) for p in table[b, : -(-n // ps)].tolist() for i in range(ps)][:n]
        if c["prefix"]:
            where = [(int(p), i) for p in s["prefix_pages"].tolist() for i in range(ps)][: c["prefix"]] + where
        pg = torch.tensor([p for p, _ in where], device=DEV)
        sl = torch.tensor([i for _, i in where], device=DEV)
        key = torch.arange(len(where), device=DEV, dtype=f64)
        for h in range(heads):
            kk, vv = s["k"][pg, h // group, sl].to(f64), s["v"][pg, h // group, sl].to(f64)
            for i0 in range(0, m, 4096):
                i1 = min(m, i0 + 4096)
                x = s["q"][t + i0: t + i1, h * hd: (h + 1) * hd].to(f64) @ kk.T / math.sqrt(hd)
                if c["cap"]:
                    x = c["cap"] * torch.tanh(x / c["cap"])
                at = torch.arange(i0, i1, device=DEV, dtype=f64)[:, None] + (c["prefix"] + n - m)
                if c["slopes"]:
                    x = x - slopes[h] * (at - key).abs()
                last = torch.clamp(at, min=c["prefix"] + c["prefix_mask"] - 1)
                x = x.masked_fill(key > last, -math.inf)
                out[t + i0: t + i1, h] = torch.softmax(x, dim=-1) @ vv
        t += m
    return out.reshape(-1, heads * hd)
