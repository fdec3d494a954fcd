"""Refusals of the entry points of a decoder's serving step: every bad argument is answered with -1 before anything is enqueued
(no GPU needed, and none is touched: refused calls only)."""
import copy
import ctypes as C
import math

import pytest

A = 0x10000      # an address that only refused calls name


def spec(odla, count=32, **kw):
    s = odla.rotary_spec([1.0 / (i + 1) for i in range(count)])
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def rotary_desc(odla, **kw):
    base = dict(dtype=1, batch=2, tokens=3, heads=4, channels=64, x_batch=768, x_token=256, x_head=64, y_batch=768, y_token=256, y_head=64)
    return odla.RotaryDesc(**dict(base, **kw))


def call_rotary(lib, s, d, x=A, y=A + 4096, pos=A):
    return lib.b200_rotary(s if s is None else C.byref(s), d if d is None else C.byref(d), x, y, pos, None)


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(dtype=-1), dict(batch=-1), dict(tokens=-2), dict(heads=-1), dict(heads=1025), dict(channels=0), dict(channels=63),
                                dict(channels=1025), dict(x_token=-1), dict(y_head=-64), dict(x_batch=1 << 50), dict(batch=1 << 16, tokens=1 << 16)])
def test_rotary_refuses_descriptors(odla, lib, kw):
    assert call_rotary(lib, spec(odla), rotary_desc(odla, **kw)) == -1


def test_rotary_refuses_pointers_and_specs(odla, lib):
    s, d = spec(odla), rotary_desc(odla)
    assert call_rotary(lib, None, d) == -1 and call_rotary(lib, s, None) == -1
    assert call_rotary(lib, s, d, x=None) == -1 and call_rotary(lib, s, d, y=None) == -1 and call_rotary(lib, s, d, pos=None) == -1
    assert call_rotary(lib, s, d, x=A + 1) == -1 and call_rotary(lib, s, d, pos=A + 2) == -1
    assert call_rotary(lib, s, rotary_desc(odla, dtype=0), x=A + 2) == -1
    assert call_rotary(lib, s, rotary_desc(odla, y_token=512), x=A, y=A) == -1        # in place with other strides
    for kw in (dict(pairs=-1), dict(pairs=129), dict(pairs=33), dict(axes=0), dict(axes=5)):
        assert call_rotary(lib, spec(odla, **kw), d) == -1
    bad = spec(odla)
    bad.axis[31] = 1
    assert call_rotary(lib, bad, d) == -1
    for f in (math.inf, -math.inf, math.nan):
        bad = spec(odla)
        bad.frequency[0] = f
        assert call_rotary(lib, bad, d) == -1
    for kw in (dict(batch=0), dict(tokens=0), dict(heads=0)):
        assert call_rotary(lib, s, rotary_desc(odla, **kw), x=None, y=None, pos=None) == 0
    with pytest.raises(ValueError):
        odla.rotary_spec([1.0] * 129)
    with pytest.raises(ValueError):
        odla.rotary_spec([1.0, 1.0], axis=[0])
    with pytest.raises(ValueError):
        odla.rotary_spec([1.0], axis=[4])


def test_rows_that_would_be_written_over_one_another_are_refused(odla, lib):
    s = spec(odla)
    for kw in (dict(y_batch=0), dict(y_token=0), dict(y_head=63), dict(y_head=1)):
        assert call_rotary(lib, s, rotary_desc(odla, **kw)) == -1, kw
    for kw in (dict(page=0), dict(head=0), dict(token=63)):
        assert call_append(lib, cache(odla, **kw), append_desc(odla), s) == -1, kw
    for kw in (dict(y_token=0), dict(y_head=32)):
        assert call_append(lib, cache(odla), append_desc(odla, **kw), s) == -1, kw
    for kw in (dict(y_batch=0), dict(y_head=56), dict(queries=2, y_token=0)):
        d = attention_desc(odla, **kw)
        assert call_attention(lib, cache(odla), d) == -1 and lib.b200_paged_attention_workspace(C.byref(cache(odla)), C.byref(d)) == -1, kw
    # a stride of an extent of one is never used, and rows that are only read may lie anywhere
    d = attention_desc(odla, batch=1, y_batch=0, y_token=0, q_head=0)
    assert lib.b200_paged_attention_workspace(C.byref(cache(odla, page=0)), C.byref(d)) > 0


def cache(odla, **kw):
    return odla.PagedCache(**dict(dict(dtype=1, pages=8, page_size=16, heads=2, channels=64, page=2048, head=1024, token=64), **kw))


def append_desc(odla, **kw):
    base = dict(tokens=3, heads=4, q_token=512, q_head=64, k_token=512, k_head=64, v_token=512, v_head=64, y_token=256, y_head=64)
    return odla.AppendDesc(**dict(base, **kw))


def call_append(lib, c, d, s, kc=A, vc=A, q=A, k=A, v=A, y=A + 64, pos=A, slots=A):
    ref = [None if x is None else C.byref(x) for x in (c, d, s)]
    return lib.b200_paged_append(ref[0], kc, vc, ref[1], ref[2], q, k, v, y, pos, slots, None)


def test_append_refuses(odla, lib):
    c, d, s = cache(odla), append_desc(odla), spec(odla)
    for kw in (dict(dtype=3), dict(pages=0), dict(page_size=0), dict(heads=0), dict(heads=2000), dict(channels=0), dict(channels=2000), dict(page=-1), dict(head=-1), dict(token=-1)):
        assert call_append(lib, cache(odla, **kw), d, s) == -1
    for kw in (dict(tokens=-1), dict(heads=-1), dict(heads=1025), dict(q_token=-1), dict(k_head=-1), dict(v_token=-1), dict(y_head=-1)):
        assert call_append(lib, c, append_desc(odla, **kw), s) == -1
    assert call_append(lib, None, d, s) == -1 and call_append(lib, c, None, s) == -1
    for name in ("kc", "vc", "q", "k", "v", "y", "pos", "slots"):
        assert call_append(lib, c, d, s, **{name: None}) == -1
        assert call_append(lib, c, d, s, **{name: A + 1}) == -1
    assert call_append(lib, c, d, s, slots=A + 4) == -1
    assert call_append(lib, c, d, s, y=A) == -1                    # in place with other strides
    assert call_append(lib, cache(odla, channels=62), d, s) == -1   # fewer channels than pairs turn
    assert call_append(lib, c, append_desc(odla, tokens=0), s, kc=None, vc=None, q=None, k=None, v=None, y=None, pos=None, slots=None) == 0


def attention_desc(odla, **kw):
    base = dict(batch=2, queries=1, heads=4, prefix_length=40, table_width=4, scale=0.125, q_batch=256, q_token=256, q_head=64, y_batch=256, y_token=256, y_head=64)
    return odla.PagedAttentionDesc(**dict(base, **kw))


def call_attention(lib, c, d, kc=A, vc=A, q=A, prefix=A, table=A, lengths=A, y=A, ws=A, size=1 << 40):
    return lib.b200_paged_attention(None if c is None else C.byref(c), kc, vc, None if d is None else C.byref(d), q, prefix, table, lengths, y, ws, size, None)


def test_attention_refuses(odla, lib):
    c, d = cache(odla), attention_desc(odla)
    need = lib.b200_paged_attention_workspace(C.byref(c), C.byref(d))
    assert need > 0
    assert call_attention(lib, c, d, size=need - 1) == -1
    bad_caches = [dict(dtype=0), dict(dtype=3), dict(channels=32), dict(channels=96), dict(channels=256), dict(token=68), dict(page=2052), dict(head=-8), dict(heads=3), dict(page_size=0)]
    bad_descs = [dict(batch=-1), dict(queries=0), dict(heads=0), dict(heads=5), dict(heads=2048), dict(prefix_length=-1), dict(table_width=-1), dict(scale=math.nan), dict(scale=math.inf),
                 dict(q_head=60), dict(y_token=-8), dict(table_width=1 << 27), dict(batch=1 << 22, queries=2)]
    for kw in bad_caches:
        x = cache(odla, **kw)
        assert lib.b200_paged_attention_workspace(C.byref(x), C.byref(d)) == -1 and call_attention(lib, x, d) == -1, kw
    for kw in bad_descs:
        x = attention_desc(odla, **kw)
        assert lib.b200_paged_attention_workspace(C.byref(c), C.byref(x)) == -1 and call_attention(lib, c, x) == -1, kw
    assert lib.b200_paged_attention_workspace(None, C.byref(d)) == -1 and call_attention(lib, None, d) == -1 and call_attention(lib, c, None) == -1
    for name in ("kc", "vc", "q", "prefix", "table", "lengths", "y", "ws"):
        assert call_attention(lib, c, d, **{name: None}) == -1, name
        assert call_attention(lib, c, d, **{name: A + 2}) == -1, name
    for name in ("kc", "vc", "q", "y", "ws"):
        assert call_attention(lib, c, d, **{name: A + 8}) == -1, name
    none = attention_desc(odla, batch=0)
    assert lib.b200_paged_attention_workspace(C.byref(c), C.byref(none)) == 0
    assert call_attention(lib, c, none, kc=None, vc=None, q=None, prefix=None, table=None, lengths=None, y=None, ws=None, size=0) == 0


def test_workspace_is_the_same_for_every_call(odla, lib):
    c, d = cache(odla), attention_desc(odla, batch=7, queries=3)
    sizes = {lib.b200_paged_attention_workspace(C.byref(copy.copy(c)), C.byref(d)) for _ in range(3)}
    assert len(sizes) == 1


def test_sample_refuses(odla, lib):
    def call(logits=A, t=A, k=A, p=A, m=A, u=A, out=A, **kw):
        d = odla.SampleDesc(**dict(dict(dtype=2, rows=4, vocab=1000, row=1000), **kw))
        return lib.b200_sample(C.byref(d), logits, t, k, p, m, u, out, None)
    for kw in (dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(rows=(1 << 24) + 1), dict(vocab=0), dict(vocab=(1 << 18) + 1), dict(row=-1), dict(logits=None), dict(u=None), dict(out=None),
               dict(logits=A + 1), dict(dtype=0, logits=A + 2), dict(t=A + 1), dict(k=A + 2), dict(p=A + 3), dict(m=A + 1), dict(u=A + 2), dict(out=A + 1)):
        assert call(**kw) == -1, kw
    assert lib.b200_sample(None, A, A, A, A, A, A, A, None) == -1
    assert call(rows=0, logits=None, u=None, out=None) == 0
