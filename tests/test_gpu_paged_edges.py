"""The paged cache's operators where their calls are at an edge: units without keys, padding, caps of every size, odd row starts."""
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
