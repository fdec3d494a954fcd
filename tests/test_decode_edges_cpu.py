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


def workspace(odla, lib, heads, channels, page, **kw):
    c = cache(odla, heads=heads[1], channels=channels, page_size=page, page=heads[1] * page * channels, head=page * channels, token=channels)
    row = heads[0] * channels
    q = kw.get("queries", 1)
    d = attention_desc(odla, **dict(dict(heads=heads[0], q_batch=q * row, q_token=row, q_head=channels, y_batch=q * row, y_token=row, y_head=channels), **kw))
    return lib.b200_paged_attention_workspace(C.byref(c), C.byref(d))


@pytest.mark.parametrize("heads,channels,page", [((32, 8), 128, 16), ((12, 12), 64, 16), ((64, 8), 128, 64), ((28, 4), 128, 24), ((8, 1), 128, 1), ((16, 2), 64, 100)])
def test_a_workspace_for_the_largest_call_serves_every_smaller_one(odla, lib, heads, channels, page):
    """Sizes never fall as batch, queries, heads, prefix or table grow: along each of them, and from any shape to any larger one."""
    import random
    batches, prefixes, widths, queries = (range(1, 200), (0, 1, 100, 129, 1999, 8192, 32768, 131072, 10 ** 6), (0, 1, 2, 5, 44, 60, 256, 1000, 8192), (1, 2, 3, 4, 5, 8, 9, 16, 17, 33, 64, 65, 70, 300))
    for prefix in prefixes:
        for width in widths:
            sizes = [workspace(odla, lib, heads, channels, page, batch=b, prefix_length=prefix, table_width=width) for b in batches]
            assert all(0 <= x <= y for x, y in zip(sizes, sizes[1:])), (prefix, width)
    rng = random.Random(heads[0] * channels + page)
    for _ in range(3000):
        large = dict(batch=rng.choice(batches), prefix_length=rng.choice(prefixes), table_width=rng.choice(widths), queries=rng.choice(queries))
        small = {k: rng.choice([v, max(v - 1, 0), v // 2, rng.randint(0, v)]) for k, v in large.items()}
        small["batch"], small["queries"] = max(small["batch"], 1), max(small["queries"], 1)
        fewer = (rng.choice([heads[0], heads[1]]), heads[1])
        assert 0 <= workspace(odla, lib, fewer, channels, page, **small) <= workspace(odla, lib, heads, channels, page, **large), (fewer, small, large)


def test_a_workspace_of_shapes_that_are_cut_finely_when_they_are_few(odla, lib):
    for prefix, own, large, small in ((0, 4096, 48, 23), (32768, 960, 100, 64), (8192, 704, 32, 30), (8192, 0, 127, 64)):
        sizes = [workspace(odla, lib, (32, 8), 128, 16, batch=b, prefix_length=prefix, table_width=own // 16) for b in (small, large)]
        assert 0 < sizes[0] <= sizes[1]


def rotary_desc(odla, **kw):
    base = dict(dtype=1, batch=2, tokens=3, heads=4, channels=64, x_batch=768, x_token=256, x_head=64, y_batch=768, y_token=256, y_head=64)
    return odla.RotaryDesc(**dict(base, **kw))


def call_rotary(odla, lib, d):
    return lib.b200_rotary(C.byref(odla.rotary_spec([0.1] * 32)), C.byref(d), A, A + 4096, A, None)


@pytest.mark.parametrize("kw", [dict(y_token=64), dict(y_token=128), dict(y_token=255), dict(y_batch=256), dict(y_batch=767), dict(y_head=300), dict(y_token=64, y_head=64, y_batch=64),
                                dict(y_head=192, y_token=64, y_batch=500)])
def test_rotary_refuses_rows_that_meet_across_strides(odla, lib, kw):
    """Each stride is above a row's channels, but rows of different tokens, heads or batch entries lie on one another, or inside one another's rows."""
    assert call_rotary(odla, lib, rotary_desc(odla, **kw)) == -1


def test_append_and_attention_refuse_rows_that_meet_across_strides(odla, lib):
    def append(c, **kw):
        d = odla.AppendDesc(**dict(dict(tokens=3, heads=4, q_token=512, q_head=64, k_token=512, k_head=64, v_token=512, v_head=64, y_token=256, y_head=64), **kw))
        return lib.b200_paged_append(C.byref(c), A, A, C.byref(d), None, A, A, A, A + 64, None, A, None)
    for kw in (dict(y_token=64), dict(y_token=192), dict(y_head=256, y_token=255), dict(y_head=256, y_token=256)):
        assert append(cache(odla), **kw) == -1, kw
    for kw in (dict(page=1024), dict(page=2040), dict(head=64, token=64), dict(head=64, token=64, page=128), dict(token=128, head=64, page=2040), dict(head=960), dict(head=1 << 20, page=1 << 20)):
        assert append(cache(odla, **kw)) == -1, kw
    for kw in (dict(y_head=256), dict(queries=3, y_batch=256), dict(queries=3, y_token=128, y_batch=768), dict(queries=3, y_token=256, y_batch=760)):
        d = attention_desc(odla, **kw)
        assert lib.b200_paged_attention_workspace(C.byref(cache(odla)), C.byref(d)) == -1 and call_attention(lib, cache(odla), d) == -1, kw


def test_layouts_of_dense_tensors_and_their_slices_are_taken(odla, lib):
    """Every order of the extents, with room between rows, and strides that no step takes."""
    import itertools
    good = [dict(y_batch=1 << 20), dict(queries=1, y_token=0), dict(batch=1, y_batch=0), dict(heads=2, y_head=128), dict(batch=2, y_batch=64, queries=3, y_token=512, y_head=128),
            dict(batch=3, y_batch=200, queries=2, y_token=5000, y_head=600)]
    for order in itertools.permutations(("y_batch", "y_token", "y_head")):
        extent, at, kw = dict(y_batch=2, y_token=5, y_head=4), 64, dict(queries=5)
        for name in order:
            kw[name] = at
            at *= extent[name]
        good.append(kw)
    for kw in good:
        assert lib.b200_paged_attention_workspace(C.byref(cache(odla)), C.byref(attention_desc(odla, **kw))) > 0, kw
    # caches are only read by attention: they may lie on one another
    assert lib.b200_paged_attention_workspace(C.byref(cache(odla, page=0, head=0, token=0)), C.byref(attention_desc(odla))) > 0


def test_offsets_that_pass_63_bits_are_refused(odla, lib):
    """No stride is too large by itself, but the last row would lie 2^60 elements or more behind the first."""
    far = 1 << 46
    assert call_rotary(odla, lib, rotary_desc(odla, batch=1, tokens=1 << 30, x_token=far)) == -1
    assert call_rotary(odla, lib, rotary_desc(odla, batch=1, tokens=1 << 30, y_token=far)) == -1
    assert call_rotary(odla, lib, rotary_desc(odla, batch=1 << 20, tokens=1 << 10, x_batch=far)) == -1

    def append(c, **kw):
        d = odla.AppendDesc(**dict(dict(tokens=1 << 20, heads=4, q_token=512, q_head=64, k_token=512, k_head=64, v_token=512, v_head=64, y_token=256, y_head=64), **kw))
        return lib.b200_paged_append(C.byref(c), A, A, C.byref(d), None, A, A, A, A + 64, None, A, None)
    for kw in (dict(q_token=far), dict(k_token=far), dict(v_token=far), dict(y_token=far)):
        assert append(cache(odla), **kw) == -1, kw
    assert append(cache(odla, pages=1 << 30, page=far)) == -1
    for c, kw in ((dict(pages=1 << 30, page=far), {}), ({}, dict(batch=1 << 20, q_batch=far)), ({}, dict(batch=1 << 20, y_batch=far)), ({}, dict(batch=1, queries=1 << 20, q_token=far))):
        d = attention_desc(odla, **kw)
        assert lib.b200_paged_attention_workspace(C.byref(cache(odla, **c)), C.byref(d)) == -1 and call_attention(lib, cache(odla, **c), d) == -1, kw
    d = odla.SampleDesc(dtype=2, rows=1 << 20, vocab=1000, row=far)
    assert lib.b200_sample(C.byref(d), A, None, None, None, None, A, A, None) == -1
