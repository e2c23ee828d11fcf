"""The paged cache's operators where their calls are at an edge: units without keys, padding, caps of every size, odd row starts."""
import ctypes
import math

import pytest
import torch

import quanta_b200 as qb
from quanta_b200 import _lib as L
from quanta_b200 import paged
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float16


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def build(m, kv_lens, ragged=True):
    cache = paged.PagedKVCache.from_parts(m["k"].to(DEV), m["v"].to(DEV))
    return cache, paged.PagedBatch(cache, m["table"].to(DEV), ints(kv_lens), ints(m["cu"]) if ragged else None)


def within(got, want, tol):
    got = got.detach().cpu().to(torch.float64)
    err = torch.where(torch.isinf(want) & (got == want), torch.zeros_like(want), (got - want).abs() - tol)
    assert not torch.isnan(got).any()
    assert (err <= 0).all(), f"off by up to {err.max():.3e} more than the bound {tol.max():.3e}"


def sees(q_lens, kv_lens):
    """Whether each token of a causal call sees a key: its place is not negative."""
    return torch.tensor([n - c + i >= 0 for c, n in zip(q_lens, kv_lens) for i in range(c)])


# (heads, K/V heads, new tokens, keys).  Tables of at most 256 keys (one page more than the longest sequence needs) are never cut into
# ranges, and more than 1024 packed rows go to the kernel for prompts: blocks of 128 rows in the first three, two tiles of 128 in the
# others (more blocks of 128 than SMs).
EMPTY = [(1, 1, [700, 400, 300], [40, 0, 200]), (6, 2, [401, 140, 60], [13, 140, 0]), (4, 1, [300, 90], [0, 90]),
         (16, 16, [700, 600, 260], [20, 0, 230]), (24, 8, [500, 513, 300], [30, 0, 200])]


@pytest.mark.parametrize("hd,dtype", [(128, BF), (64, FP)])
@pytest.mark.parametrize("heads,kv_heads,q_lens,kv_lens", EMPTY)
def test_blocks_of_a_prompt_that_see_no_key(heads, kv_heads, q_lens, kv_lens, hd, dtype):
    """More new tokens than keys: zeros and -inf wherever no key is seen, in every one of many calls, whatever Q holds."""
    m = ref.make(17, q_lens, kv_lens, heads, kv_heads, hd, 16, dtype)
    cache, batch = build(m, kv_lens)
    q = m["q"].to(DEV)
    some = sees(q_lens, kv_lens).to(DEV)
    first = None
    for i in range(12):
        out = torch.full_like(q, 77.0)
        lse = torch.full((q.shape[0], heads), 77.0, device=DEV)
        paged.paged_attention(batch, q, out=out, lse=lse)
        assert (out[~some] == 0.0).all() and (lse[~some] == -math.inf).all()
        if first is None:
            first = out, lse
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])
    cache.check()
    # the definition, at the first and last rows that see something
    at = some.cpu().nonzero().flatten()
    at = at[:1].tolist() + at[-1:].tolist()
    want, wl, tol, ltol = ref.attention(m["q"], m["k"], m["v"], m["table"], kv_lens, m["cu"], heads, 1.0 / math.sqrt(hd))
    within(first[0][at], want[at], tol[at])
    within(first[1][at], wl[at], ltol[at])


@pytest.mark.parametrize("heads,kv_heads,q_lens,kv_lens", [EMPTY[0], EMPTY[1], EMPTY[4]])
def test_blocks_that_see_only_a_shared_prefix(heads, kv_heads, q_lens, kv_lens):
    """Rows without keys of their own behind a prefix: the prefix's result alone, the same as without any own keys."""
    prefix = 23
    m = ref.make(18, q_lens, kv_lens, heads, kv_heads, 128, 16, BF, prefix=prefix)
    cache, batch = build(m, kv_lens)
    q, pages = m["q"].to(DEV), m["pre"].to(DEV)
    none = ~sees(q_lens, kv_lens).to(DEV)
    bare = paged.PagedBatch(cache, batch.table, torch.zeros_like(batch.kv_lens), batch.cu_q)
    alone, l0 = torch.empty_like(q), torch.empty(q.shape[0], heads, device=DEV)
    paged.shared_prefix_attention(bare, q, pages, prefix, out=alone, lse=l0)
    for _ in range(8):
        out, lse = torch.full_like(q, 77.0), torch.full((q.shape[0], heads), 77.0, device=DEV)
        paged.shared_prefix_attention(batch, q, pages, prefix, out=out, lse=lse)
        assert torch.equal(out[none], alone[none]) and torch.equal(lse[none], l0[none])
    cache.check()
    want, wl, tol, ltol = ref.attention(m["q"][:1], m["k"], m["v"], m["table"], [0], [0, 1], heads, 1.0 / math.sqrt(128), prefix=(m["pre"], prefix))
    within(alone[:1], want, tol)
    within(l0[:1], wl, ltol)


@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (6, 2)])
def test_ranges_without_keys(heads, kv_heads):
    """A short prompt in a table that could hold 40000 keys is cut into ten ranges, most of them empty; calls with narrow tables
    between such calls keep their bits, and so do they."""
    q_lens, kv_lens = [300, 70], [310, 70]
    m = ref.make(19, q_lens, kv_lens, heads, kv_heads, 128, 16, BF, width=2500)
    cache, batch = build(m, kv_lens)
    q = m["q"].to(DEV)
    tight = paged.PagedBatch(cache, batch.table[:, :20].contiguous(), batch.kv_lens, batch.cu_q)
    a, b = paged.paged_attention(batch, q), paged.paged_attention(tight, q)
    scratch = torch.full((batch._floats[(q.shape[0], heads)],), float("nan"), device=DEV)
    for _ in range(8):
        scratch.fill_(float("nan"))  # what an empty range does not write is not used
        assert torch.equal(paged.paged_attention(batch, q, scratch=scratch), a)
        assert torch.equal(paged.paged_attention(tight, q), b)
    cache.check()
    want, _, tol, _ = ref.attention(m["q"], m["k"], m["v"], m["table"], kv_lens, m["cu"], heads, 1.0 / math.sqrt(128))
    within(a, want, tol)
    within(b, want, tol)


@pytest.fixture()
def no_patience():
    lib = L.load()
    assert lib.qb200_paged_set_spin_limit(1) == 0
    yield lib
    assert lib.qb200_paged_set_spin_limit(4 << 20) == 0


def test_spin_limit_setter_rejects_zero():
    assert L.load().qb200_paged_set_spin_limit(0) == L.ERR_INVALID_PARAM and "positive" in L.last_error()


# one tile of rows and two, keys in one range and in several, Q by boxes and row by row, behind a prefix
@pytest.mark.parametrize("heads,kv_heads,q_lens,hd,dtype,width,prefix", [
    (8, 2, [300, 70], 128, BF, 0, 0), (8, 2, [300, 70], 64, FP, 2500, 0), (6, 2, [400, 1], 128, BF, 0, 0), (16, 16, [700, 500, 300], 64, FP, 0, 0),
    (24, 8, [500, 513], 128, BF, 0, 0), (8, 2, [300, 70], 128, BF, 0, 700)])
def test_waits_that_run_out_are_reported(no_patience, heads, kv_heads, q_lens, hd, dtype, width, prefix):
    """With a single poll per wait the kernel gives up wherever a copy or a product is not there yet: it returns, the status says
    so once, and the next calls are as they were."""
    lib = no_patience
    kv_lens = [n + 5 for n in q_lens]
    m = ref.make(23, q_lens, kv_lens, heads, kv_heads, hd, 16, dtype, prefix=prefix, width=width)
    cache, batch = build(m, kv_lens)
    q, pages = m["q"].to(DEV), m["pre"].to(DEV)

    def call():
        return paged.shared_prefix_attention(batch, q, pages, prefix) if prefix else paged.paged_attention(batch, q)

    lib.qb200_paged_set_spin_limit(4 << 20)
    want = call()
    cache.check()
    ran_out = 0
    for _ in range(5):
        lib.qb200_paged_set_spin_limit(1)
        got = call()
        try:
            cache.check()
            assert torch.equal(got, want)
        except qb.QuantError as e:
            assert e.code == L.ERR_TIMEOUT and "wait ran out" in str(e)
            ran_out += 1
        cache.check()  # reported once
        lib.qb200_paged_set_spin_limit(4 << 20)
        assert torch.equal(call(), want)
        cache.check()
    assert ran_out


def capped(m, kv_lens, heads, cap, scale, prefix=0):
    """The definition in float64 with caps of any size: (out, bound of |out - exact|), causal.

    The bound is that of paged_reference.attention but for the cap, whose error is relative to the score, not to the cap: with
    x = score / cap, below |x| = 0.3 a polynomial of relative error 2e-6 at most (its best fit's 1.9e-6, four roundings), above it
    1 - 2 / (e^2x + 1) of absolute error 2^-21 (exponential 2^-22, half of it reaches the result; reciprocal, sums 2^-23 each), which is 1.7e-6 of
    tanh(0.3): below 2^-18 |score| in all."""
    hd, kvh = m["k"].shape[3], m["k"].shape[1]
    group, u, dt = heads // kvh, ref.HALF_STEP[m["k"].dtype], m["k"].dtype
    q = m["q"].to(ref.F64).reshape(-1, heads, hd)
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    pre = [ref.keys_of(p, m["pre"], prefix) for p in (m["k"], m["v"])]
    for b, n in enumerate(kv_lens):
        kk, vv = (torch.cat([x, ref.keys_of(p, m["table"][b], n)], 1) for x, p in zip(pre, (m["k"], m["v"])))
        lo, hi = m["cu"][b], m["cu"][b + 1]
        for t in range(lo, hi):
            see = prefix + n - (hi - lo) + (t - lo) + 1
            for h in range(heads):
                K, V = kk[h // group, :see], vv[h // group, :see]
                s = K @ q[t, h] * scale
                e = float((hd + 8) * 2.0 ** -24 * abs(scale) * (K.abs() @ q[t, h].abs()).max())
                s = cap * torch.tanh(s / cap)
                e += float((2.0 ** -18 + 2.0 ** -21) * s.abs().max())
                p = torch.softmax(s, 0)
                out[t, h] = p @ V
                A = p @ V.abs()
                tol[t, h] = u * out[t, h].abs() + (u + 2 * e + 2 * (see / 16 + 64) * 2.0 ** -24 + 2.0 ** -20) * (1 + u) * A
                if dt == FP:
                    tol[t, h] += see * 2.0 ** -25 * V.abs().max() + 2.0 ** -25
    return out.reshape(-1, heads * hd), tol.reshape(-1, heads * hd)


@pytest.mark.parametrize("cap", [1e-6, 0.5, 30.0, 1e3, 1e5, 1e6, 1e8, 1e20])
@pytest.mark.parametrize("q_lens,kv_lens,heads,prefix", [([1, 1, 1], [40, 1, 300], 4, 0), ([3, 1], [9, 170], 4, 70), ([270, 3], [270, 90], 8, 0)])
def test_caps_of_every_size(q_lens, kv_lens, heads, prefix, cap):
    """A cap far above the scores leaves them as they are, in the kernels for few rows as in the one for prompts."""
    for hd, dtype, scale, width in ((128, BF, None, 0), (64, FP, 0.4, 2500)):
        m = ref.make(29, q_lens, kv_lens, heads, 2, hd, 16, dtype, prefix=prefix, width=width)
        cache, batch = build(m, kv_lens)
        q = m["q"].to(DEV)
        if prefix:
            out = paged.shared_prefix_attention(batch, q, m["pre"].to(DEV), prefix, scale=scale, softcap=cap)
        else:
            out = paged.paged_attention(batch, q, scale=scale, softcap=cap)
        cache.check()
        within(out, *capped(m, kv_lens, heads, cap, 1.0 / math.sqrt(hd) if scale is None else scale, prefix))


@pytest.mark.parametrize("cap", [2e30, 1e38, 3.4e38])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [40, 300]), ([270, 3], [270, 90])])
def test_the_largest_caps(q_lens, kv_lens, cap):
    """Near the end of the 32-bit range the cap does nothing."""
    m = ref.make(30, q_lens, kv_lens, 8, 2, 128, 16, BF)
    cache, batch = build(m, kv_lens)
    q = m["q"].to(DEV)
    assert torch.equal(paged.paged_attention(batch, q, softcap=cap), paged.paged_attention(batch, q))
    cache.check()


@pytest.mark.parametrize("width", [0, 2500])
def test_no_tokens_behind_a_shared_prefix(width):
    m = ref.make(33, [0, 0], [20, 9], 4, 2, 128, 16, BF, prefix=40, width=width)
    cache, batch = build(m, [20, 9])
    q = torch.empty(0, 512, dtype=BF, device=DEV)
    assert paged.shared_prefix_attention(batch, q, m["pre"].to(DEV), 40).shape == (0, 512)
    cache.check()


def test_workspace_sizes_of_refused_calls():
    """0 and a message, whatever the descriptions hold; nothing is read through their pointers."""
    lib, P = L.load(), 1 << 20
    good, seqs = dict(n_pages=10, page_size=16, kv_heads=2, head_dim=128, dtype=L.BF16), dict(table_stride=8, table_width=8, batch=3)

    def sizes(kv=(), b=(), tokens=5, heads=4, prefix=20):
        c = L.PagedKv(k_pages=P, v_pages=P, status_dev=P, **{**good, **dict(kv)})
        s = L.PagedBatch(table=P, kv_lens=P, cu_q=P, **{**seqs, **dict(b)})
        c, s = ctypes.byref(c), ctypes.byref(s)
        return lib.qb200_paged_attention_scratch_floats(c, s, tokens, heads), lib.qb200_shared_prefix_scratch_floats(c, s, prefix, tokens, heads)

    assert sizes()[1] > 0
    assert sizes(b=dict(table_width=2500, table_stride=2500), tokens=1000)[0] > 0  # keys cut into ranges
    for kw in (dict(b=dict(batch=0)), dict(b=dict(table_width=0)), dict(b=dict(table_stride=7)), dict(b=dict(table_width=1 << 28, table_stride=1 << 28)),
               dict(kv=dict(page_size=0)), dict(kv=dict(page_size=48)), dict(kv=dict(page_size=0xFFFFFFFF)), dict(kv=dict(kv_heads=0)), dict(kv=dict(head_dim=0)),
               dict(kv=dict(n_pages=0)), dict(kv=dict(dtype=L.F32)), dict(heads=0), dict(heads=3), dict(tokens=1 << 28), dict(tokens=1 << 27, heads=64)):
        assert sizes(**kw) == (0, 0), kw
        assert "scratch_floats" in L.last_error()
    for n in (0, 1 << 31, (1 << 31) - 128, (1 << 64) - 1):
        assert sizes(prefix=n)[1] == 0, n
        assert "qb200_shared_prefix_scratch_floats" in L.last_error()
    assert lib.qb200_paged_attention_scratch_floats(None, None, 5, 4) == 0 and lib.qb200_shared_prefix_scratch_floats(None, None, 20, 5, 4) == 0


@pytest.mark.parametrize("q_lens", [[3, 1], [200, 130]])
@pytest.mark.parametrize("before", [1, 5, 150])
def test_rows_before_the_first_sequence(q_lens, before):
    """cu_q that does not begin at 0: the rows before it belong to nobody, in append as in both attentions, and nothing is reported."""
    heads, kvh, hd, prefix, kv_lens = 8, 2, 128, 50, [n + 20 for n in q_lens]
    m = ref.make(35, q_lens, kv_lens, heads, kvh, hd, 16, BF, garbage=0.5, prefix=prefix)
    cache, batch = build(m, kv_lens)
    rows, a, c = m["cu"][-1], heads * hd, (heads + kvh) * hd
    x = torch.randn(before + rows + 2, (heads + 2 * kvh) * hd, generator=torch.Generator().manual_seed(1)).to(BF).to(DEV)
    y = x[before: before + rows]
    late = paged.PagedBatch(cache, batch.table, batch.kv_lens, batch.cu_q + before)
    cos, sin = paged.rope_table(400, hd, device=DEV)
    own = slice(before, before + rows)

    def left(t):
        return (t[:before] == 77.0).all() and (t[before + rows:] == 77.0).all()

    q = paged.paged_rope_append(batch, y[:, :a], y[:, a:c], y[:, c:], cos, sin)
    k, v = cache.k.clone(), cache.v.clone()
    cache.k.copy_(m["k"])
    cache.v.copy_(m["v"])
    q2 = torch.full((x.shape[0], a), 77.0, dtype=BF, device=DEV)
    paged.paged_rope_append(late, x[:, :a], x[:, a:c], x[:, c:], cos, sin, q_out=q2)
    cache.check()
    assert torch.equal(q2[own], q) and left(q2) and torch.equal(cache.k, k) and torch.equal(cache.v, v)
    for call in (lambda b, q, **kw: paged.paged_attention(b, q, **kw), lambda b, q, **kw: paged.shared_prefix_attention(b, q, m["pre"].to(DEV), prefix, **kw)):
        out, lse = torch.full_like(q2, 77.0), torch.full((x.shape[0], heads), 77.0, device=DEV)
        call(late, q2, out=out, lse=lse)
        cache.check()
        want = call(batch, q)
        # (the other row of a tile, and the other number of rows, may change how a row's keys are cut and joined)
        assert ((out[own].double() - want.double()).abs() <= 4 * 2.0 ** -8 * float(v.float().abs().max())).all()
        assert left(out) and left(lse)
    cache.check()


@pytest.mark.parametrize("kw", [dict(), dict(softcap=40.0), dict(softcap=1e4)], ids=str)
@pytest.mark.parametrize("heads,kv_heads,hd,dtype", [(4, 4, 128, BF), (8, 2, 64, FP), (6, 2, 128, BF)])
def test_rows_of_nobody_and_of_others_change_no_bit(heads, kv_heads, hd, dtype, kw):
    """A padded batch: the rows behind the last sequence hold anything, and so do the next sequence's; both share tiles with the
    rows before them."""
    q_lens, kv_lens, tail = [300, 77, 300], [333, 90, 300], 60
    m = ref.make(37, q_lens, kv_lens, heads, kv_heads, hd, 16, dtype, tail=tail)
    cache, batch = build(m, kv_lens)
    q = m["q"].to(DEV) * 0.5
    rows, first = sum(q_lens), q_lens[0]
    want = paged.paged_attention(batch, q, **kw)
    for junk in (float("nan"), float("inf"), 300.0, 0.0):
        q[rows:] = junk
        assert torch.equal(paged.paged_attention(batch, q, **kw)[:rows], want[:rows]), junk
    for junk in (float("nan"), 300.0, 0.0):
        q[first: first + q_lens[1]] = junk
        got = paged.paged_attention(batch, q, **kw)
        assert torch.equal(got[:first], want[:first]) and torch.equal(got[first + q_lens[1]: rows], want[first + q_lens[1]: rows]), junk
    cache.check()


@pytest.mark.parametrize("dtype,hd", [(BF, 128), (FP, 128), (BF, 64), (FP, 64)])
@pytest.mark.parametrize("width", [0, 2500])
def test_weights_of_tokens_are_not_rounded_to_the_type(dtype, hd, width):
    """Few rows: the softmax weights enter the second product as a sum of two numbers of the cache's type.

    The bound is that of paged_reference.attention with u A, the rounding of the weights to the type, replaced by that of the
    second part: half a step of at most half a step, u^2 A (f16: the second part's smallest step is there already, n 2^-25 max |v|)."""
    heads, kvh, scale = 8, 2, 0.01  # scores near 0: even weights, and little error from the scores themselves
    q_lens, kv_lens = [1, 1, 2, 1, 3], [7, 12, 30, 65, 11]
    m = ref.make(41, q_lens, kv_lens, heads, kvh, hd, 16, dtype, width=width)
    cache, batch = build(m, kv_lens)
    out = paged.paged_attention(batch, m["q"].to(DEV), scale=scale)
    cache.check()
    want, _, tol, _ = ref.attention(m["q"], m["k"], m["v"], m["table"], kv_lens, m["cu"], heads, scale)
    mags = dict(m, v=m["v"].abs())
    A = ref.attention(mags["q"], mags["k"], mags["v"], mags["table"], kv_lens, mags["cu"], heads, scale)[0]  # sum of p |v|
    u = ref.HALF_STEP[dtype]
    within(out, want, tol - (u - u * u) * (1 + u) * A)


@pytest.mark.parametrize("width", [40, 2500])
def test_captured_prompts_follow_row_starts_and_lengths(width):
    """A padded, captured step of append, attention and attention behind a prefix, replayed with other sequences: prompts where tokens
    were, none at all, more new tokens than keys."""
    heads, kvh, hd, ps, B, rows, prefix = 8, 2, 128, 16, 3, 420, 50
    m = ref.make(43, [0] * B, [600] * B, heads, kvh, hd, ps, BF, garbage=0.5, prefix=prefix, width=width)
    cache, _ = build(m, [600] * B)
    kv, cu = ints([1, 1, 1]), ints([0, 1, 2, 3])
    batch = paged.PagedBatch(cache, m["table"].to(DEV), kv, cu)
    cos, sin = paged.rope_table(700, hd, device=DEV)
    x = torch.randn(rows, (heads + 2 * kvh) * hd, device=DEV).to(BF)
    a, b, pre = heads * hd, (heads + kvh) * hd, m["pre"].to(DEV)

    def step():
        q = paged.paged_rope_append(batch, x[:, :a], x[:, a:b], x[:, b:], cos, sin)
        return q, paged.paged_attention(batch, q), paged.shared_prefix_attention(batch, q, pre, prefix)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for q_lens, kv_lens in (([1, 1, 1], [5, 600, 90]), ([300, 1, 100], [300, 20, 500]), ([0, 0, 0], [7, 0, 600]), ([1, 419, 0], [0, 30, 9]), ([140, 140, 140], [140, 600, 300])):
        c = [0]
        for n in q_lens:
            c.append(c[-1] + n)
        kv.copy_(ints(kv_lens))
        cu.copy_(ints(c))
        x.copy_(torch.randn_like(x))
        g.replay()
        want = step()
        for w, r in zip(want, got):
            assert torch.equal(w[: c[-1]], r[: c[-1]])
    cache.check()
