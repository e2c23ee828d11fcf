"""Refusals of the paged cache's entry points (no GPU: every check below comes before the first CUDA call), its Python
checks, and the table of angles."""
import ctypes

import numpy as np
import pytest
import torch

import quanta_b200 as qb
from quanta_b200 import _lib as L
from quanta_b200 import paged
from quanta_b200.decoder import rope_rows

lib = L.load()
P = 1 << 20  # an aligned address that is never read


def kv(**kw):
    d = dict(k_pages=P, v_pages=P, status_dev=P, n_pages=10, page_size=16, kv_heads=2, head_dim=128, dtype=L.BF16)
    d.update(kw)
    return L.PagedKv(**d)


def seqs(**kw):
    d = dict(table=P, kv_lens=P, cu_q=P, table_stride=8, table_width=8, batch=3)
    d.update(kw)
    return L.PagedBatch(**d)


def attend(c=None, b=None, q=P, q_stride=512, tokens=5, heads=4, scale=0.1, cap=0.0, scratch=P, out=2 * P):
    return lib.qb200_paged_attention(ctypes.byref(c or kv()), ctypes.byref(b or seqs()), q, q_stride, tokens, heads, scale, cap, None, None, 1, scratch, out, None, None)


def prefix(c=None, b=None, pages=P, n=20, q=P, tokens=5, heads=4, cap=0.0, out=2 * P):
    return lib.qb200_shared_prefix_attention(ctypes.byref(c or kv()), ctypes.byref(b or seqs()), pages, n, q, 512, tokens, heads, 0.1, cap, None, P, out, None, None)


def append(c=None, b=None, q=P, k=P, v=P, dt=L.F32, qs=512, ks=256, vs=256, tokens=5, heads=4, cos=P, sin=P, rot=128, n_pos=9, q_out=P):
    return lib.qb200_paged_rope_append(ctypes.byref(c or kv()), ctypes.byref(b or seqs()), q, k, v, dt, qs, ks, vs, tokens, heads, cos, sin, rot, n_pos, None, q_out, None)


CACHE = [(dict(k_pages=None), 8), (dict(v_pages=None), 8), (dict(status_dev=None), 8), (dict(k_pages=P + 8), 8), (dict(dtype=L.F32), 5), (dict(head_dim=96), 5),
         (dict(page_size=8), 5), (dict(page_size=48), 5), (dict(page_size=512), 5), (dict(page_size=0), 5), (dict(kv_heads=0), 8), (dict(n_pages=0), 8),
         (dict(n_pages=1 << 31), 8)]
BATCH = [(dict(table=None), 8), (dict(kv_lens=None), 8), (dict(batch=0), 8), (dict(table_width=0), 7), (dict(table_stride=7), 7),
         (dict(table_width=1 << 28, table_stride=1 << 28), 5), (dict(cu_q=None), 7)]


@pytest.mark.parametrize("call", [attend, prefix, append])
def test_every_entry_point_checks_the_cache_and_the_batch(call):
    for kw, code in CACHE:
        assert call(c=kv(**kw)) == code, kw
        assert "qb200_" in L.last_error()
    for kw, code in BATCH:
        assert call(b=seqs(**kw)) == code, kw


def test_attention_refusals():
    for f in (attend, prefix):
        assert f(heads=3) == L.ERR_INVALID_PARAM and "multiple" in L.last_error()
        assert f(heads=0) == L.ERR_INVALID_PARAM
        assert f(q=None) == L.ERR_INVALID_PARAM
        assert f(q=P + 2) == L.ERR_INVALID_PARAM and f(out=P) == L.ERR_INVALID_PARAM
        assert f(cap=-1.0) == L.ERR_INVALID_PARAM and f(cap=float("inf")) == L.ERR_INVALID_PARAM and f(cap=1e-9) == L.ERR_INVALID_PARAM
        assert f(tokens=1 << 28) == L.ERR_NOT_SUPPORTED
    assert attend(q_stride=500) == L.ERR_LENGTH and attend(q_stride=516) == L.ERR_LENGTH
    assert attend(scale=float("nan")) == L.ERR_INVALID_PARAM
    assert attend(out=None) == L.ERR_INVALID_PARAM and attend(scratch=P + 4) == L.ERR_INVALID_PARAM and attend(out=P + 4) == L.ERR_INVALID_PARAM
    assert prefix(n=0) == L.ERR_INVALID_PARAM and prefix(pages=None) == L.ERR_INVALID_PARAM and prefix(n=1 << 31) == L.ERR_NOT_SUPPORTED
    assert attend(tokens=0) == L.OK and prefix(tokens=0) == L.OK  # nothing to do


def test_append_refusals():
    assert append(dt=7) == L.ERR_NOT_SUPPORTED
    for kw in (dict(k=None), dict(v=None), dict(cos=None), dict(sin=None), dict(q=None), dict(q_out=None), dict(rot=0), dict(rot=130), dict(rot=7), dict(n_pos=0),
               dict(q_out=P + 8), dict(k=P + 2)):
        assert append(**kw) == L.ERR_INVALID_PARAM, kw
    for kw in (dict(qs=511), dict(ks=255), dict(vs=0)):
        assert append(**kw) == L.ERR_LENGTH, kw
    assert append(tokens=0) == L.OK


def test_python_refusals():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    good = paged.PagedKVCache.from_parts(k, k.clone())
    for bad in (lambda: paged.PagedKVCache.from_parts(k, k[:3]), lambda: paged.PagedKVCache.from_parts(k.float(), k.float()),
                lambda: paged.PagedKVCache.from_parts(k.transpose(1, 2), k.transpose(1, 2)), lambda: paged.PagedKVCache.from_parts(k, k.half()),
                lambda: paged.PagedKVCache(4, 24, 2, 64, device="cpu"), lambda: paged.PagedKVCache(4, 16, 2, 80, device="cpu"),
                lambda: paged.PagedKVCache(0, 16, 2, 64, device="cpu")):
        with pytest.raises(qb.QuantError):
            bad()
    t, n = torch.zeros(3, 4, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    cu = torch.arange(4, dtype=torch.int32)
    paged.PagedBatch(good, t, n, cu)
    for args in ((t.long(), n, cu), (t, n.long(), cu), (t, n, cu[:3]), (t, n[:2], cu), (t.t(), n, cu), (t[:, :0], n, cu), (t[:1].expand(3, 4), n, cu), (t[0], n, cu)):
        with pytest.raises(qb.QuantError):
            paged.PagedBatch(good, *args)


def test_angles_are_those_of_the_single_position_rows():
    cos, sin = paged.rope_table(300, 128, device="cpu")
    assert cos.shape == sin.shape == (300, 64)
    for pos in (0, 1, 257, 299):
        c, s = rope_rows(pos, 128)
        assert np.array_equal(cos[pos].numpy(), c[:64]) and np.array_equal(sin[pos].numpy(), s[:64])
