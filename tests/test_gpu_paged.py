"""The paged cache's operators on the GPU against their definitions in float64 (tests/paged_reference.py)."""
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


# A table that could hold this many pages a sequence: the lengths' upper bound is what decides which kernel a call takes, so
# short sequences in wide tables reach the kernels that long ones would.
WIDE = 2500


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def build(m, kv_lens, ragged=True):
    cache = paged.PagedKVCache.from_parts(m["k"].to(DEV), m["v"].to(DEV))
    return cache, paged.PagedBatch(cache, m["table"].to(DEV), ints(kv_lens), ints(m["cu"]) if ragged else None)


def within(got, want, tol, rows=None):
    got = got.detach().cpu().to(torch.float64)
    if rows is not None:
        got, want, tol = got[:rows], want[:rows], tol[:rows]
    same = torch.isinf(want) & (got == want)
    err = torch.where(same, torch.zeros_like(want), (got - want).abs() - tol)
    assert not torch.isnan(got).any()
    assert (err <= 0).all(), f"off by up to {err.max():.3e} more than the bound {tol.max():.3e}"


def run(seed, q_lens, kv_lens, heads, kv_heads, hd=128, ps=16, dtype=BF, tail=0, prefix=0, cap=0.0, slopes=False, prefix_lens=None, causal=True, scale=None,
        ragged=True, garbage=float("nan"), width=0):
    m = ref.make(seed, q_lens, kv_lens, heads, kv_heads, hd, ps, dtype, garbage, prefix, tail=tail, width=width)
    sc = 1.0 / math.sqrt(hd) if scale is None else scale
    sl = torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32) if slopes else None
    cache, batch = build(m, kv_lens, ragged)
    rows = m["cu"][-1]
    q = m["q"].to(DEV)
    out = torch.full_like(q, 77.0)
    lse = torch.full((q.shape[0], heads), 77.0, device=DEV)
    sd = None if sl is None else sl.to(DEV)
    if prefix:
        got = paged.shared_prefix_attention(batch, q, m["pre"].to(DEV), prefix, scale=scale, softcap=cap, slopes=sd, out=out, lse=lse)
    else:
        got = paged.paged_attention(batch, q, scale=scale, softcap=cap, slopes=sd, prefix_lens=None if prefix_lens is None else ints(prefix_lens), causal=causal,
                                    out=out, lse=lse)
    assert got is out
    cache.check()
    want, wl, tol, ltol = ref.attention(m["q"], m["k"], m["v"], m["table"], kv_lens, m["cu"], heads, sc, cap, sl, prefix_lens, causal,
                                        (m["pre"], prefix) if prefix else None)
    within(out, want, tol, rows)
    within(lse, wl, ltol, rows)
    assert (out[rows:] == 77.0).all() and (lse[rows:] == 77.0).all()  # rows behind the last sequence
    return m, cache, batch, out


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 2), (7, 1), (20, 1), (40, 1)])
def test_single_tokens(heads, kv_heads, dtype, hd):
    """One new token per sequence, from one key to several tiles, with and without explicit row starts."""
    kv = [1, 2, 15, 16, 17, 63, 64, 65, 130, 257]
    for width in (0, WIDE):
        run(heads + hd, [1] * len(kv), kv, heads, kv_heads, hd, 16, dtype, ragged=False, width=width)
    run(heads + hd + 1, [1] * len(kv), kv, heads, kv_heads, hd, 32, dtype, tail=3)


@pytest.mark.parametrize("width", [0, WIDE])
@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256])
def test_page_sizes(ps, width):
    run(ps, [1, 1, 1, 5], [ps - 1, ps, ps + 1, 3 * ps + 7], 8, 2, ps=ps, width=width)
    run(ps + 1, [70, 33], [ps + 70, 333], 8, 2, ps=ps, dtype=FP, hd=64, width=width)


@pytest.mark.parametrize("dtype,hd", [(BF, 128), (FP, 128), (BF, 64), (FP, 64)])
@pytest.mark.parametrize("heads,kv_heads,q_lens,kv_lens", [
    (2, 2, [1, 17, 130, 300], [1, 17, 130, 300]),        # whole prompts
    (8, 2, [64, 1, 5, 2], [200, 90, 5, 400]),            # chunks, single tokens, drafts
    (6, 2, [129, 43], [129, 500]),                       # a group that does not divide a tile
    (4, 1, [256, 257], [256, 600]),
])
def test_prompts(heads, kv_heads, q_lens, kv_lens, dtype, hd):
    for width in (0, WIDE):
        run(len(q_lens) * 7 + heads, q_lens, kv_lens, heads, kv_heads, hd, 16, dtype, tail=5, width=width)


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [40, 90, 300]), ([100, 3, 1], [180, 90, 300]), ([200, 200], [200, 261])])
@pytest.mark.parametrize("kw", [dict(cap=3.0), dict(slopes=True), dict(cap=20.0, slopes=True), dict(prefix_lens=[60, 0, 1000]), dict(causal=False),
                                dict(causal=False, slopes=True), dict(scale=0.5), dict(scale=0.0), dict(scale=-0.1, cap=2.0)], ids=str)
def test_scores_and_masks(q_lens, kv_lens, kw):
    kw = dict(kw)
    if "prefix_lens" in kw:
        kw["prefix_lens"] = kw["prefix_lens"][: len(q_lens)]
    for width in (0, WIDE):
        run(31, q_lens, kv_lens, 4, 2, 128, 16, BF, width=width, **kw)
        run(32, q_lens, kv_lens, 6, 2, 64, 32, FP, width=width, **kw)


def test_rows_and_sequences_that_see_nothing():
    """No keys at all, more new tokens than keys, no new tokens: zeros and -inf where nothing is seen."""
    for width in (0, WIDE):
        run(5, [1, 1, 1], [0, 3, 0], 4, 2, ragged=False, width=width)
        run(6, [3, 0, 5, 1, 0], [0, 9, 2, 0, 0], 4, 2, tail=2, width=width)
        run(7, [200, 0, 3], [140, 50, 0], 4, 2, width=width)
        run(8, [1, 130], [0, 5], 8, 1, prefix=19, width=width)


@pytest.mark.parametrize("hd,dtype", [(64, FP), (128, BF)])
def test_prompts_of_many_tiles_in_one_block(hd, dtype):
    """Enough blocks for every SM, so that one takes all its keys: the ring of tiles goes round several times, and the last
    tile's unused rows (NaN here) are cleared in the right turn of it."""
    run(3, [260] * 5, [900, 1000, 1111, 260, 1290], 8, 8, hd, 16, dtype, width=WIDE)
    run(4, [130] * 10, [600 + 37 * i for i in range(10)], 8, 8, hd, 64, dtype, width=WIDE, cap=9.0)


def wide_run(q_lens, kv_lens, heads, kv_heads, hd, dtype, ps=16, width=4096, **kw):
    """As run(), with a table far wider than the sequences need: the lengths' upper bound decides how the work is cut."""
    m = ref.make(77, q_lens, kv_lens, heads, kv_heads, hd, ps, dtype)
    cache = paged.PagedKVCache.from_parts(m["k"].to(DEV), m["v"].to(DEV))
    table = torch.full((len(kv_lens), width), -3, dtype=torch.int32)
    table[:, : m["table"].shape[1]] = m["table"]
    batch = paged.PagedBatch(cache, table.to(DEV), ints(kv_lens), ints(m["cu"]))
    out = paged.paged_attention(batch, m["q"].to(DEV), **kw)
    cache.check()
    want, _, tol, _ = ref.attention(m["q"], m["k"], m["v"], m["table"], kv_lens, m["cu"], heads, 1.0 / math.sqrt(hd), kw.get("softcap", 0.0))
    within(out, want, tol)


@pytest.mark.parametrize("hd,dtype", [(128, BF), (64, FP)])
def test_many_short_sequences_in_wide_tables(hd, dtype):
    """Several units in one CTA's run, units cut by run ends, more sequences than a CTA keeps lengths of, empty ones between."""
    g = torch.Generator().manual_seed(3)
    kv = torch.randint(1, 200, (170,), generator=g).tolist()
    q = [1] * 170
    for i in (0, 17, 127, 128, 129, 169):
        q[i] = kv[i] = 0
    for i in (5, 60, 140):
        q[i] = min(3, kv[i])
    wide_run(q, kv, 8, 4, hd, dtype)
    wide_run([1, 1, 0, 1], [2900, 1, 40, 700], 4, 1, hd, dtype)
    wide_run([1], [1], 4, 4, hd, dtype, softcap=2.0)


def test_more_sequences_than_a_block_has_threads():
    """Prompts among many single tokens: the prompt kernel's search over a long batch."""
    q, kv = [1] * 430, [1 + i % 7 for i in range(430)]
    for i, (a, b) in {3: (40, 50), 200: (0, 0), 399: (70, 70), 400: (33, 90), 429: (20, 20)}.items():
        q[i], kv[i] = a, b
    run(13, q, kv, 2, 1, 64, 16, FP)


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [700, 90]), ([300], [700])])
@pytest.mark.parametrize("width", [0, WIDE])
@pytest.mark.parametrize("rising", [True, False])
def test_scores_that_rise_and_fall_along_the_keys(q_lens, kv_lens, rising, width):
    """The running maximum moves in every tile, or never after the first; scores of several hundred, one key wins."""
    m = ref.make(5, q_lens, kv_lens, 2, 1, 128, 16, BF, width=width)
    for b, n in enumerate(kv_lens):
        for j in range(n):
            x = (j if rising else n - j) / n
            m["k"][int(m["table"][b, j // 16]), :, j % 16] = (m["k"][int(m["table"][b, j // 16]), :, j % 16].float() * 0.05 + 4.0 * x).to(BF)
    m["q"] = (m["q"].float().abs() + 0.5).to(BF)
    cache, batch = build(m, kv_lens)
    out = paged.paged_attention(batch, m["q"].to(DEV))
    cache.check()
    want, _, tol, _ = ref.attention(m["q"], m["k"], m["v"], m["table"], kv_lens, m["cu"], 2, 1.0 / math.sqrt(128))
    within(out, want, tol)


def test_two_calls_at_once():
    """Prompts and single tokens over the same cache and batch from two streams."""
    m = ref.make(90, [260, 1, 30], [600, 900, 200], 8, 2, 128, 16, BF, garbage=0.25)
    cache, batch = build(m, [600, 900, 200])
    ones = paged.PagedBatch(cache, batch.table, batch.kv_lens)
    q, q1 = m["q"].to(DEV), torch.randn(3, 1024, device=DEV).to(BF)
    want, want1 = paged.paged_attention(batch, q), paged.paged_attention(ones, q1)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    a.wait_stream(torch.cuda.current_stream())
    b.wait_stream(torch.cuda.current_stream())
    got, got1 = [], []
    for _ in range(20):
        with torch.cuda.stream(a):
            got.append(paged.paged_attention(batch, q))
        with torch.cuda.stream(b):
            got1.append(paged.paged_attention(ones, q1))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got) and all(torch.equal(x, want1) for x in got1)
    cache.check()


def test_long_keys_and_few_sequences():
    """One sequence over every SM: its keys are cut into many runs that are joined."""
    run(9, [1], [5003], 4, 2, ragged=False)
    run(10, [2, 1], [3001, 1], 3, 1, hd=64, dtype=FP)
    run(11, [40], [2500], 4, 1)
    run(12, [3, 1], [10, 9000], 40, 1)


@pytest.mark.parametrize("prefix", [1, 16, 100, 333])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1, 1], [1, 9, 70, 33]), ([3, 1, 40], [3, 9, 140]), ([1] * 20, list(range(1, 21))), ([150], [200]), ([290, 1], [300, 20])])
def test_shared_prefix(prefix, q_lens, kv_lens):
    for width in (0, WIDE):
        run(prefix, q_lens, kv_lens, 8, 2, prefix=prefix, tail=1, width=width)
        run(prefix + 1, q_lens, kv_lens, 3, 3, hd=64, ps=32, dtype=FP, prefix=prefix, cap=5.0, slopes=True, width=width)


def test_shared_prefix_long():
    """A prefix that one row's share of CTAs cuts into ranges, for few rows and for many."""
    run(71, [1, 1], [5, 40], 8, 2, prefix=5000)
    run(72, [1, 2], [5, 40], 3, 1, prefix=4100, hd=64, dtype=FP, slopes=True)
    run(73, [60, 1], [60, 3], 40, 2, prefix=700)


def test_shared_prefix_equals_attention_over_the_whole_sequence():
    """The same keys once behind a shared prefix and once as plain sequences that name the prefix's pages first."""
    heads, kvh, hd, ps, prefix, kv = 8, 4, 128, 16, 96, [5, 40, 17]
    m = ref.make(3, [1, 1, 1], kv, heads, kvh, hd, ps, BF, prefix=prefix)
    cache, batch = build(m, kv, ragged=False)
    q = m["q"].to(DEV)
    got = paged.shared_prefix_attention(batch, q, m["pre"].to(DEV), prefix)
    table = torch.cat([m["pre"][None].expand(3, -1), m["table"]], 1).contiguous().to(DEV)
    whole = paged.paged_attention(paged.PagedBatch(cache, table, ints([n + prefix for n in kv])), q)
    # both lie within their bounds of the same numbers: half a step for the result and half a step for the weights each
    sel = m["k"].isnan().logical_not()
    vmax = float(m["v"][sel].abs().max())
    assert ((got.double() - whole.double()).abs() <= 4 * 2.0 ** -8 * vmax).all()
    cache.check()


@pytest.mark.parametrize("src,dtype", [(torch.float32, BF), (BF, BF), (FP, FP), (torch.float32, FP), (FP, BF)])
@pytest.mark.parametrize("hd,rot", [(128, 128), (64, 64), (128, 64), (64, 16), (128, 6), (64, 2)])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [1, 16, 40]), ([5, 0, 33, 2], [5, 7, 50, 19])])
def test_append(src, dtype, hd, rot, q_lens, kv_lens):
    heads, kvh, ps = 6, 2, 16
    m = ref.make(1, q_lens, kv_lens, heads, kvh, hd, ps, dtype, garbage=3.0)
    cache, batch = build(m, kv_lens, ragged=max(q_lens) > 1 or min(q_lens) < 1)
    T, tail = m["cu"][-1], 2 if batch.cu_q is not None else 0
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(T + tail, (heads + 2 * kvh) * hd, generator=g).to(src)
    a, b = heads * hd, (heads + kvh) * hd
    dq = qkv.to(DEV)
    cos, sin = paged.rope_table(64, rot, device=DEV)
    places = torch.cat([torch.arange(n - c, n) for c, n in zip(q_lens, kv_lens)])
    seqs = torch.cat([torch.full((c,), i, dtype=torch.int64) for i, c in enumerate(q_lens)])
    for positions in (None, ((places * 3 + 5) % 64)):
        pos = places if positions is None else positions
        dpos = None if positions is None else torch.cat([pos, torch.zeros(tail, dtype=torch.int64)]).to(torch.int32).to(DEV)
        q_out = torch.full((T + tail, a), 55.0, dtype=dtype, device=DEV)
        got = paged.paged_rope_append(batch, dq[:, :a], dq[:, a:b], dq[:, b:], cos, sin, positions=dpos, q_out=q_out)
        cache.check()
        assert got is q_out and (q_out[T:] == 55.0).all()
        cc, ss = cos.cpu()[pos], sin.cpu()[pos]
        u = ref.HALF_STEP[dtype]
        tiny = 2.0 ** -25 if dtype == FP else 0.0
        for x, where in ((qkv[:T, :a].double().reshape(T, heads, hd), q_out[:T].reshape(T, heads, hd).cpu()), (qkv[:T, a:b].double().reshape(T, kvh, hd), None)):
            want, e = ref.rotate(x, cc, ss)
            if where is None:
                where = cache.k.cpu()[m["table"].long()[seqs, places // ps], :, places % ps]
            within(where, want, (u * want.abs() + e) * (1 + u) + tiny)
        vv = cache.v.cpu()[m["table"].long()[seqs, places // ps], :, places % ps]
        assert torch.equal(vv, qkv[:T, b:].to(dtype).reshape(T, kvh, hd))
        # nothing else was touched
        for pool, was in ((cache.k.cpu().clone(), m["k"]), (cache.v.cpu().clone(), m["v"])):
            pool[m["table"].long()[seqs, places // ps], :, places % ps] = was[m["table"].long()[seqs, places // ps], :, places % ps]
            assert torch.equal(pool, was)
    # keys and values alone
    before = cache.k.clone()
    assert paged.paged_rope_append(batch, None, dq[:, a:b], dq[:, b:], cos, sin, positions=dpos) is None
    assert torch.equal(before, cache.k)
    cache.check()


@pytest.mark.parametrize("src", [torch.float32, BF])
def test_append_many_tokens_and_unaligned_rows(src):
    """A prompt of thousands of tokens; the same rows at odd addresses (one element at a time) give the same bits."""
    heads, kvh, hd, ps, T = 4, 2, 64, 32, 2501
    table = torch.randperm(90, generator=torch.Generator().manual_seed(1)).to(torch.int32).reshape(1, 90).to(DEV)
    w = (heads + 2 * kvh) * hd
    x = torch.randn(T, w, generator=torch.Generator().manual_seed(2)).to(src).to(DEV)
    odd = torch.empty(T, w + 3, dtype=src, device=DEV)
    odd[:, 1: 1 + w] = x
    odd = odd[:, 1: 1 + w]
    cos, sin = paged.rope_table(T + 9, hd, device=DEV)
    a, b = heads * hd, (heads + kvh) * hd
    got = []
    for y in (x, odd):
        cache = paged.PagedKVCache(90, ps, kvh, hd, device=DEV)
        batch = paged.PagedBatch(cache, table, ints([T + 4]), ints([0, T]))
        got.append((paged.paged_rope_append(batch, y[:, :a], y[:, a:b], y[:, b:], cos, sin), cache.k, cache.v))
        cache.check()
    assert all(torch.equal(p, q) for p, q in zip(*got))
    places = torch.arange(4, T + 4)
    want, e = ref.rotate(x[:, :a].cpu().double().reshape(T, heads, hd), cos.cpu()[places], sin.cpu()[places])
    within(got[0][0].reshape(T, heads, hd), want, (2.0 ** -8 * want.abs() + e) * (1 + 2.0 ** -8))
    page, slot = table.cpu()[0, places // ps].long(), places % ps
    assert torch.equal(got[0][2].cpu()[page, :, slot].reshape(T, -1), x[:, b:].cpu().to(BF))


def test_append_rotates_as_the_single_position_kernel_does():
    """Against decoder.rope_append at one position: the same products, at most one rounding apart."""
    from quanta_b200 import decoder as dec
    b, heads, hd, pos = 5, 4, 128, 37
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(b, heads * hd, generator=g).to(DEV) for _ in range(3))
    c, s = dec.rope_rows(pos, hd)
    kc = torch.zeros(b, 64, heads, hd, dtype=BF, device=DEV)
    vc, q_old = torch.zeros_like(kc), torch.empty(b, heads * hd, dtype=BF, device=DEV)
    dec.rope_append(q, k, v, torch.from_numpy(c).to(DEV), torch.from_numpy(s).to(DEV), heads, q_old, kc, vc, pos)
    cache = paged.PagedKVCache(b * 4, 16, heads, hd, device=DEV)
    table = torch.arange(b * 4, dtype=torch.int32, device=DEV).reshape(b, 4)
    batch = paged.PagedBatch(cache, table, ints([pos + 1] * b))
    q_new = paged.paged_rope_append(batch, q, k, v, *paged.rope_table(64, hd, device=DEV))
    # equal up to one rounding of a sum whose last bit may differ between a fused and an unfused product
    assert ((q_new.double() - q_old.double()).abs() <= 2 * 2.0 ** -8 * q_old.double().abs() + 2.0 ** -20).all()
    assert torch.equal(cache.v[table[:, pos // 16].long(), :, pos % 16], vc[:, pos])


def test_strided_queries():
    heads, hd, kv = 4, 128, [20, 70, 3]
    m = ref.make(12, [1, 1, 1], kv, heads, 2, hd, 16, BF)
    cache, batch = build(m, kv, ragged=False)
    wide = torch.randn(3, heads * hd + 264, device=DEV).to(BF)
    wide[:, 136: 136 + heads * hd] = m["q"].to(DEV)
    got = paged.paged_attention(batch, wide[:, 136: 136 + heads * hd])
    assert torch.equal(got, paged.paged_attention(batch, m["q"].to(DEV)))
    one = paged.PagedBatch(cache, batch.table[:1], batch.kv_lens[:1])
    odd = torch.randn(1, heads * hd + 1, device=DEV).to(BF)[:, : heads * hd]  # a single row, whatever its stride
    assert torch.equal(paged.paged_attention(one, odd), paged.paged_attention(one, odd.contiguous()))
    # a table that is a window of a wider one
    t = torch.full((3, 40), -1, dtype=torch.int32, device=DEV)
    t[:, 4: 4 + m["table"].shape[1]] = m["table"].to(DEV)
    b2 = paged.PagedBatch(cache, t[:, 4: 4 + m["table"].shape[1]], ints(kv))
    assert torch.equal(got, paged.paged_attention(b2, m["q"].to(DEV)))


def test_graph_follows_lengths_and_pages():
    """A captured step (append, attention, attention behind a prefix) follows the lengths and pages of its replay, and two
    captured steps do not disturb one another."""
    heads, kvh, hd, ps, B, prefix = 8, 2, 128, 16, 4, 40
    m = ref.make(21, [1] * B, [90] * B, heads, kvh, hd, ps, BF, garbage=0.5, prefix=prefix)
    cache, _ = build(m, [90] * B, ragged=False)
    kv = ints([3, 20, 64, 90])
    table = m["table"].to(DEV)
    batch = paged.PagedBatch(cache, table, kv)
    cos, sin = paged.rope_table(128, hd, device=DEV)
    x = torch.randn(B, (heads + 2 * kvh) * hd, device=DEV)
    a, b = heads * hd, (heads + kvh) * hd
    pre = m["pre"].to(DEV)

    def step():
        q = paged.paged_rope_append(batch, x[:, :a], x[:, a:b], x[:, b:], cos, sin)
        return paged.paged_attention(batch, q), paged.shared_prefix_attention(batch, q, pre, prefix)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = step()
    with torch.cuda.graph(g2):
        o2 = step()
    for lens in ([3, 20, 64, 90], [50, 1, 80, 17], [16, 33, 2, 49]):
        kv.copy_(ints(lens))
        x.copy_(torch.randn_like(x))
        g1.replay()
        g2.replay()
        want = step()
        for w, p, r in zip(want, o1, o2):
            assert torch.equal(w, p) and torch.equal(w, r)
    cache.check()


def test_other_stream_and_repeatability():
    m, cache, batch, out = run(41, [1, 30, 300], [700, 330, 300], 8, 2)
    q = m["q"].to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            assert torch.equal(paged.paged_attention(batch, q), out)
    side.synchronize()


@pytest.mark.parametrize("width", [0, WIDE])
def test_calls_from_new_threads(width):
    """A thread whose first CUDA work this is, three at a time."""
    import threading
    m, cache, batch, out = run(91, [300, 1], [300, 90], 8, 2, width=width)
    q, seen = m["q"].to(DEV), []
    torch.cuda.synchronize()

    def work():
        try:
            seen.append(all(torch.equal(paged.paged_attention(batch, q), out) for _ in range(10)))
        except Exception as e:
            seen.append(e)

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert seen == [True] * 3
    cache.check()


@pytest.mark.parametrize("kw", [dict(), dict(cap=20.0), dict(slopes=True), dict(cap=20.0, slopes=True)], ids=str)
def test_results_do_not_depend_on_what_ran_before(kw):
    """The same call gives the same bits whatever other calls left in the SMs' shared memory: the last tile of a sequence
    holds rows that nothing was copied to."""
    q_lens = kv_lens = [469, 300, 77]
    m, cache, batch, out = run(55, q_lens, kv_lens, 2, 1, 128, 16, BF, **kw)
    sl = torch.tensor([2.0 ** (-4.0 * (h + 1)) for h in range(2)], device=DEV) if kw.get("slopes") else None
    loud = ref.make(56, q_lens, [512, 384, 128], 2, 1, 128, 16, BF)
    loud_cache = paged.PagedKVCache.from_parts((loud["k"] * 40).to(DEV), loud["v"].to(DEV))
    loud_batch = paged.PagedBatch(loud_cache, loud["table"].to(DEV), ints([512, 384, 128]), ints(loud["cu"]))
    q = m["q"].to(DEV)
    for _ in range(4):
        paged.paged_attention(loud_batch, loud["q"].to(DEV))
        assert torch.equal(paged.paged_attention(batch, q, softcap=kw.get("cap", 0.0), slopes=sl), out)
        quiet = paged.PagedBatch(loud_cache, loud_batch.table, ints([0, 0, 0]), loud_batch.cu_q)
        paged.paged_attention(quiet, loud["q"].to(DEV))
        assert torch.equal(paged.paged_attention(batch, q, softcap=kw.get("cap", 0.0), slopes=sl), out)


def test_what_the_host_cannot_see_is_reported():
    heads, hd, kv = 4, 128, [20, 70, 3]
    m = ref.make(50, [1, 1, 1], kv, heads, 2, hd, 16, BF, garbage=0.0)
    cache, batch = build(m, kv, ragged=False)
    q = m["q"].to(DEV)
    good = paged.paged_attention(batch, q)
    for bad in (-1, cache.n_pages, 2 ** 31 - 1, -2 ** 31):  # page numbers outside the pool
        t = m["table"].clone()
        t[1, 2] = bad
        got = paged.paged_attention(paged.PagedBatch(cache, t.to(DEV), ints(kv)), q)
        with pytest.raises(qb.QuantError) as e:
            cache.check()
        assert e.value.kind == "InvalidParam"
        cache.check()  # reported once
        assert torch.equal(got[0], good[0]) and torch.equal(got[2], good[2])  # the other sequences are as they were
    for lens in ([20, 10 ** 6, 3], [20, -5, 3]):  # more keys than the table holds; a negative length
        t = m["table"].clone().clamp(min=0)
        got = paged.paged_attention(paged.PagedBatch(cache, t.to(DEV), ints(lens)), q)
        with pytest.raises(qb.QuantError) as e:
            cache.check()
        assert e.value.kind == "LengthMismatch"
        assert torch.equal(got[0], good[0]) and torch.equal(got[2], good[2])
    for cu in ([0, 2, 1, 3], [0, 1, 2, 9], [-4, 1, 2, 3]):
        paged.paged_attention(paged.PagedBatch(cache, m["table"].to(DEV), ints(kv), ints(cu)), q)
        with pytest.raises(qb.QuantError):
            cache.check()
    # append: a bad page and a place behind the table write nothing; a position outside the angles is reported
    k0, v0 = cache.k.clone(), cache.v.clone()
    cos, sin = paged.rope_table(128, hd, device=DEV)
    x = torch.randn(3, 2 * hd, device=DEV)
    for t, lens in ((torch.full_like(m["table"], -1), kv), (m["table"], [10 ** 6] * 3)):
        paged.paged_rope_append(paged.PagedBatch(cache, t.to(DEV), ints(lens)), None, x, x, cos, sin, positions=ints([0, 0, 0]))
        with pytest.raises(qb.QuantError):
            cache.check()
        assert torch.equal(cache.k, k0) and torch.equal(cache.v, v0)
    for p in ([0, 128, 0], [0, -1, 0]):
        paged.paged_rope_append(batch, None, x, x, cos, sin, positions=ints(p))
        with pytest.raises(qb.QuantError):
            cache.check()


def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements, with the used pages at its far end."""
    heads, kvh, hd, ps = 8, 8, 128, 64
    n_pages = (1 << 32) // (kvh * ps * hd) + 9
    k = torch.empty(n_pages, kvh, ps, hd, dtype=BF, device=DEV)
    v = torch.empty_like(k)
    kv = [150, 100]
    m = ref.make(60, [1, 70], kv, heads, kvh, hd, ps, BF, garbage=0.0)
    n = m["k"].shape[0]
    k[-n:], v[-n:] = m["k"].to(DEV), m["v"].to(DEV)
    cache = paged.PagedKVCache.from_parts(k, v)
    table = torch.where(m["table"] >= 0, m["table"] + (n_pages - n), m["table"])
    batch = paged.PagedBatch(cache, table.to(DEV), ints(kv), ints(m["cu"]))
    x = torch.randn(71, kvh * hd, device=DEV)
    paged.paged_rope_append(batch, None, x, x, *paged.rope_table(200, hd, device=DEV))
    small = paged.PagedKVCache.from_parts(k[-n:].clone(), v[-n:].clone())
    got = paged.paged_attention(batch, m["q"].to(DEV))
    want = paged.paged_attention(paged.PagedBatch(small, m["table"].to(DEV), ints(kv), ints(m["cu"])), m["q"].to(DEV))
    assert torch.equal(got, want)
    assert torch.equal(cache.v[table[0, 149 // ps].long(), :, 149 % ps].reshape(-1), x[0].to(BF))
    cache.check()


def test_a_serving_run():
    """Prompts, then decode steps behind them, through append and attention: every step equals the definition over the
    whole sequence as the cache holds it."""
    heads, kvh, hd, ps = 4, 2, 64, 16
    cache = paged.PagedKVCache(24, ps, kvh, hd, device=DEV)
    cache.k.fill_(float("nan"))
    cache.v.fill_(float("nan"))
    table = torch.arange(24, dtype=torch.int32, device=DEV).reshape(3, 8)
    cos, sin = paged.rope_table(128, hd, device=DEV)
    kv = [0, 0, 0]
    g = torch.Generator().manual_seed(8)
    for q_lens in ([37, 5, 64], [1, 1, 1], [1, 0, 1], [4, 2, 1], [20, 1, 0]):
        kv = [n + c for n, c in zip(kv, q_lens)]
        cu = [0]
        for c in q_lens:
            cu.append(cu[-1] + c)
        x = torch.randn(cu[-1], (heads + 2 * kvh) * hd, generator=g).to(BF).to(DEV)
        batch = paged.PagedBatch(cache, table, ints(kv), ints(cu))
        a, b = heads * hd, (heads + kvh) * hd
        q = paged.paged_rope_append(batch, x[:, :a], x[:, a:b], x[:, b:], cos, sin)
        out = paged.paged_attention(batch, q)
        cache.check()
        want, _, tol, _ = ref.attention(q.cpu(), cache.k.cpu(), cache.v.cpu(), table.cpu(), kv, cu, heads, 1.0 / math.sqrt(hd))
        within(out, want, tol)


def test_python_refusals_on_the_device():
    m = ref.make(70, [1, 1], [20, 9], 4, 2, 128, 16, BF)
    cache, batch = build(m, [20, 9], ragged=False)
    q = m["q"].to(DEV)
    one = torch.ones(4, device=DEV)
    for call in (lambda: paged.paged_attention(batch, q.to(FP)), lambda: paged.paged_attention(batch, q[:1]), lambda: paged.paged_attention(batch, q[:, :384]),
                 lambda: paged.paged_attention(batch, q[:, :500]), lambda: paged.paged_attention(batch, q.cpu()),
                 lambda: paged.paged_attention(batch, q, softcap=-1.0), lambda: paged.paged_attention(batch, q, scale=float("nan")),
                 lambda: paged.paged_attention(batch, q, slopes=one[:3]), lambda: paged.paged_attention(batch, q, slopes=one.double()),
                 lambda: paged.paged_attention(batch, q, prefix_lens=ints([1])), lambda: paged.paged_attention(batch, q, out=q[:1]),
                 lambda: paged.paged_attention(batch, q, lse=one), lambda: paged.paged_attention(batch, q, scratch=one.double()),
                 lambda: paged.shared_prefix_attention(batch, q, ints([1]), 16, scratch=one),
                 lambda: paged.shared_prefix_attention(batch, q, ints([1]), 17), lambda: paged.shared_prefix_attention(batch, q, ints([1]), 0),
                 lambda: paged.paged_rope_append(batch, q, q[:, :256], q[:, :128], one, one),
                 lambda: paged.paged_rope_append(batch, q, q[:, :256], q[:, :256], one.reshape(2, 2), one.reshape(1, 4)),
                 lambda: paged.paged_rope_append(batch, q, q[:, :256].float(), q[:, :256], one.reshape(2, 2), one.reshape(2, 2)),
                 lambda: paged.paged_rope_append(batch, None, q[:, :256], q[:, :256], torch.ones(2, 80, device=DEV), torch.ones(2, 80, device=DEV))):
        with pytest.raises(qb.QuantError):
            call()
    assert paged.paged_attention(paged.PagedBatch(cache, batch.table, batch.kv_lens, ints([0, 0, 0])), q[:0]).shape == (0, 512)
    cache.check()
