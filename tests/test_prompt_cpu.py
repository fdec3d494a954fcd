"""Refusals of the norm, of attention of a chunk and of log probabilities: every bad argument is answered with -1 before anything is enqueued (no GPU
needed, and none is touched: refused calls only)."""
import ctypes as C
import math

import pytest

A = 0x100000      # an address that only refused calls name


def norm(odla, lib, x=A, r=A * 2, w=A * 3, s=A * 4, y=A * 5, q=A * 6, scales=A * 7, **kw):
    base = dict(dtype=1, weight_dtype=0, rows=3, heads=2, channels=64, quant=1, group=32, epsilon=1e-5, weight_offset=0.0, x_row=256, x_head=64, residual_row=128, residual_head=64, sum_row=128,
                sum_head=64, y_row=128, y_head=64, quant_row=128, quant_head=64)
    return lib.b200_rms_norm(C.byref(odla.RmsNormDesc(**dict(base, **kw))), x, r, w, s, y, q, scales, None)


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(dtype=-1), dict(weight_dtype=3), dict(weight_dtype=-1), dict(rows=-1), dict(heads=-1), dict(heads=1025), dict(channels=0), dict(channels=32769),
                                dict(quant=3), dict(quant=-1), dict(group=-1), dict(group=48), dict(group=4), dict(group=128), dict(epsilon=-1.0), dict(epsilon=math.nan), dict(epsilon=math.inf),
                                dict(weight_offset=math.nan), dict(x_row=-1), dict(residual_head=-1), dict(sum_row=-1), dict(y_head=-1), dict(quant_row=-1), dict(x_row=1 << 50),
                                dict(rows=1 << 30, heads=2), dict(rows=(1 << 31) - 1, heads=1024), dict(sum_row=64), dict(y_head=63), dict(quant_row=0), dict(quant_head=32)])
def test_norm_refuses_descriptors(odla, lib, kw):
    assert norm(odla, lib, **kw) == -1


@pytest.mark.parametrize("kw", [dict(x=None), dict(x=A + 1), dict(r=None), dict(r=A + 1), dict(w=A + 2), dict(s=A + 1), dict(y=A + 1), dict(q=None), dict(scales=None), dict(scales=A + 2),
                                dict(quant=0), dict(s=None, y=None, q=None, quant=0), dict(r=None, s=A), dict(dtype=0, x=A + 2), dict(weight_dtype=1, w=A + 1),
                                dict(s=A, sum_row=128), dict(y=A), dict(y=A * 2, y_row=256), dict(q=A), dict(q=A * 2), dict(s=A * 5), dict(q=A * 4), dict(q=A * 5)])
def test_norm_refuses_pointers(odla, lib, kw):
    """Missing, unaligned, or results over one another; in place with other strides."""
    assert norm(odla, lib, **kw) == -1


def test_norm_of_nothing_is_a_call(odla, lib):
    assert lib.b200_rms_norm(None, A, A, A, A, A, A, A, None) == -1
    none = dict(x=None, r=None, w=None, s=None, y=None, q=None, scales=None)
    assert norm(odla, lib, rows=0, **none) == 0 and norm(odla, lib, heads=0, **none) == 0


def cache(odla, **kw):
    return odla.PagedCache(**dict(dict(dtype=1, pages=8, page_size=16, heads=2, channels=64, page=2048, head=1024, token=64), **kw))


def chunk(odla, lib, c=None, kc=A, vc=A, q=A, starts=A, prefix=A, table=A, lengths=A, y=A * 2, **kw):
    base = dict(batch=2, tokens=9, heads=4, prefix_length=40, table_width=4, scale=0.125, q_token=256, q_head=64, y_token=256, y_head=64)
    return lib.b200_chunk_attention(C.byref(cache(odla) if c is None else c), kc, vc, C.byref(odla.ChunkAttentionDesc(**dict(base, **kw))), q, starts, prefix, table, lengths, y, None)


@pytest.mark.parametrize("kw", [dict(dtype=0), dict(dtype=3), dict(channels=32), dict(channels=96), dict(channels=256), dict(token=68), dict(page=2052), dict(head=-8), dict(heads=3),
                                dict(page_size=0), dict(pages=0), dict(heads=0)])
def test_chunk_refuses_caches(odla, lib, kw):
    assert chunk(odla, lib, c=cache(odla, **kw)) == -1


@pytest.mark.parametrize("kw", [dict(batch=-1), dict(batch=1 << 20), dict(tokens=-1), dict(tokens=1 << 24), dict(tokens=1 << 23, heads=64), dict(heads=0), dict(heads=5), dict(heads=2048), dict(prefix_length=-1),
                                dict(table_width=-1), dict(scale=math.nan), dict(scale=math.inf), dict(q_head=60), dict(q_token=-8), dict(y_token=-8), dict(y_token=128), dict(y_head=32),
                                dict(table_width=1 << 27), dict(prefix_length=1 << 30), dict(y=A), dict(kc=None), dict(vc=None), dict(q=None), dict(starts=None), dict(prefix=None), dict(table=None),
                                dict(lengths=None), dict(y=None), dict(kc=A + 8), dict(vc=A + 8), dict(q=A + 8), dict(y=A + 8), dict(starts=A + 2), dict(prefix=A + 2), dict(table=A + 1), dict(lengths=A + 3)])
def test_chunk_refuses(odla, lib, kw):
    if kw == dict(y=A):
        kw = dict(y=A, y_token=512)                # in place with other strides
    assert chunk(odla, lib, **kw) == -1


def test_chunk_of_nothing_is_a_call(odla, lib):
    none = dict(kc=None, vc=None, q=None, starts=None, prefix=None, table=None, lengths=None, y=None)
    assert chunk(odla, lib, batch=0, **none) == 0 and chunk(odla, lib, tokens=0, **none) == 0
    assert lib.b200_chunk_attention(C.byref(cache(odla)), A, A, None, A, A, A, A, A, A, None) == -1
    d = odla.ChunkAttentionDesc(batch=1, tokens=1, heads=1)
    assert lib.b200_chunk_attention(None, A, A, C.byref(d), A, A, A, A, A, A, None) == -1


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(rows=(1 << 24) + 1), dict(vocab=0), dict(vocab=(1 << 18) + 1), dict(given=-1), dict(given=(1 << 18) + 1), dict(top=-1),
                                dict(top=65), dict(row=-1), dict(row=1 << 47), dict(l=None), dict(l=A + 1), dict(dtype=0, l=A + 2), dict(t=A + 1), dict(tokens=None), dict(lp=None), dict(tokens=A + 2),
                                dict(lp=A + 1), dict(e=A + 2), dict(tt=None), dict(tl=None), dict(tt=A + 1), dict(tl=A + 2)])
def test_log_probs_refuses(odla, lib, kw):
    p = dict(l=A, t=A, tokens=A, lp=A, e=A, tt=A, tl=A)
    p.update({k: v for k, v in kw.items() if k in p})
    d = odla.LogProbsDesc(**dict(dict(dtype=2, rows=4, vocab=1000, given=2, top=5, row=1000), **{k: v for k, v in kw.items() if k not in p}))
    assert lib.b200_log_probs(C.byref(d), p["l"], p["t"], p["tokens"], p["lp"], p["e"], p["tt"], p["tl"], None) == -1


def test_log_probs_of_nothing_is_a_call(odla, lib):
    assert lib.b200_log_probs(None, A, A, A, A, A, A, A, None) == -1
    assert lib.b200_log_probs(C.byref(odla.LogProbsDesc(dtype=0, rows=0, vocab=10, given=1, top=1, row=10)), None, None, None, None, None, None, None, None) == 0
