"""Refusals of the paged cache's entry points for arguments at the ends of their ranges (no GPU: every check comes before the first
CUDA call)."""
import ctypes

import pytest

from quanta_b200 import _lib as L

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


def attention_size(c=None, b=None, tokens=5, heads=4):
    return lib.qb200_paged_attention_scratch_floats(ctypes.byref(c or kv()), ctypes.byref(b or seqs()), tokens, heads)


def prefix_size(c=None, b=None, n=20, tokens=5, heads=4):
    return lib.qb200_shared_prefix_scratch_floats(ctypes.byref(c or kv()), ctypes.byref(b or seqs()), n, tokens, heads)


@pytest.mark.parametrize("size,name", [(attention_size, "qb200_paged_attention_scratch_floats"), (prefix_size, "qb200_shared_prefix_scratch_floats")])
def test_workspace_sizes_say_why_they_are_none(size, name):
    for kw in (dict(b=seqs(batch=0)), dict(b=seqs(table_width=0)), dict(c=kv(page_size=0xFFFFFFFF)), dict(c=kv(page_size=48)), dict(c=kv(kv_heads=0)),
               dict(c=kv(head_dim=0)), dict(heads=0), dict(heads=3), dict(tokens=1 << 28)):
        assert size(**kw) == 0, kw
        assert L.last_error().startswith(name), kw


def test_prefixes_past_the_range():
    for n in (0, 1 << 31, (1 << 31) - 128, (1 << 64) - 1):
        assert prefix_size(n=n) == 0
        assert L.last_error().startswith("qb200_shared_prefix_scratch_floats"), n


def test_tiles_of_a_prefix_are_counted_in_32_bits():
    """All K/V heads' tiles of 64 keys: refused from 2^32 on, as a table's are."""
    c = kv(kv_heads=1024)

    def call(n):
        return lib.qb200_shared_prefix_attention(ctypes.byref(c), ctypes.byref(seqs()), P, n, P, 1024 * 128, 5, 1024, 0.1, 0.0, None, None, 2 * P, None, None)

    assert call(1 << 28) == L.ERR_NOT_SUPPORTED and "2^32 tiles" in L.last_error()
    assert call((1 << 28) - 63) == L.ERR_NOT_SUPPORTED and "2^32 tiles" in L.last_error()
    assert "2^32 tiles" not in (call((1 << 28) - 64), L.last_error())[1]  # one tile a head fewer
