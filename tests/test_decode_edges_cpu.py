"""Arguments at the edges of what a decoder's entry points allow: refused calls and sizes only (no GPU needed, and none is touched)."""
import ctypes as C

import pytest

A = 0x10000      # an address that only refused calls name


def cache(odla, **kw):
    return odla.PagedCache(**dict(dict(dtype=1, pages=8, page_size=16, heads=2, channels=64, page=2048, head=1024, token=64), **kw))


def attention_desc(odla, **kw):
    base = dict(batch=2, queries=1, heads=4, prefix_length=40, table_width=4, scale=0.125, q_batch=256, q_token=256, q_head=64, y_batch=256, y_token=256, y_head=64)
    return odla.PagedAttentionDesc(**dict(base, **kw))


def call_attention(lib, c, d, size=1 << 62):
    return lib.b200_paged_attention(C.byref(c), A, A, C.byref(d), A, A, A, A, A, A, size, None)


@pytest.mark.parametrize("batch,queries,heads", [(1 << 27, 1 << 27, 1 << 10), (1 << 30, 1 << 30, 16), (1 << 22, 1 << 20, 4), (1 << 24, 1, 2), (1 << 22, 1, 4), (1, 1 << 24, 2)])
def test_attention_refuses_more_rows_than_it_counts(odla, lib, batch, queries, heads):
    """batch * queries * heads is bounded whatever its size: products of three ints that pass 64 bits, and are zero modulo 2^64, too."""
    for table_width, prefix_length in ((4, 40), (0, 40), (0, 0)):
        d = attention_desc(odla, batch=batch, queries=queries, heads=heads, table_width=table_width, prefix_length=prefix_length,
                           q_token=64 * heads, q_batch=64 * heads, y_token=64 * heads, y_batch=64 * heads * queries)
        assert lib.b200_paged_attention_workspace(C.byref(cache(odla)), C.byref(d)) == -1
        assert call_attention(lib, cache(odla), d) == -1
