"""Rotation, paged append, paged attention and sampling through the C ABI against plain 64-bit forms."""
import ctypes as C

import numpy as np
import pytest
import torch

import decode_ref as R

pytestmark = pytest.mark.gpu


def gen(*seed):
    return torch.Generator(device="cuda").manual_seed(hash(seed) % (1 << 31))


def randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(R.TORCH[dtype])


def freqs(pairs, base=10000.0):
    return [base ** (-i / max(pairs, 1)) for i in range(pairs)]


# ------------------------------------------------------------------------ rotary ----
@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("batch,tokens,heads,channels,pairs,axes", [(1, 1, 1, 2, 1, 1), (2, 5, 3, 64, 32, 2), (1, 37, 12, 128, 64, 3), (3, 17, 2, 80, 24, 1), (1, 4, 1, 7, 3, 4),
                                                                    (1, 300, 4, 256, 128, 3), (2, 3, 5, 16, 0, 1), (1, 1000, 1, 32, 16, 1),
                                                                    (1, 3, 2, 1023, 100, 1), (1, 2500, 7, 64, 32, 2)])
def test_rotary(odla, gpu_lib, dtype, interleaved, batch, tokens, heads, channels, pairs, axes):
    g = gen(dtype, tokens, channels)
    x = randn(g, (batch, tokens, heads, channels), dtype)
    pos = torch.randint(-5, 1 << 20, (axes, batch, tokens), generator=g, device="cuda", dtype=torch.int32)
    axis = [i * axes // max(pairs, 1) for i in range(pairs)]
    f = [(-1) ** (i % 3 == 2) * v for i, v in enumerate(freqs(pairs))]
    s = odla.rotary_spec(f, axis=axis, interleaved=interleaved)
    s.axes = axes
    want, size = R.turned(x, pos, f, axis, interleaved)
    for heads_first, in_place, pad in ((False, False, 0), (True, False, 0), (False, True, 0), (False, False, 3), (True, True, 8)):
        shape = (batch, heads, tokens, channels + pad) if heads_first else (batch, tokens, heads, channels + pad)
        src = torch.full(shape, 9.0, dtype=x.dtype, device="cuda")
        view = src[..., :channels].transpose(1, 2) if heads_first else src[..., :channels]
        view.copy_(x)
        dst = src if in_place else torch.full_like(src, 9.0)
        out = dst[..., :channels].transpose(1, 2) if heads_first else dst[..., :channels]
        d = odla.RotaryDesc(dtype=dtype, batch=batch, tokens=tokens, heads=heads, channels=channels, x_batch=view.stride(0), x_token=view.stride(1), x_head=view.stride(2),
                            y_batch=out.stride(0), y_token=out.stride(1), y_head=out.stride(2))
        assert gpu_lib.b200_rotary(C.byref(s), C.byref(d), src.data_ptr(), dst.data_ptr(), pos.data_ptr(), R.stream()) == 0
        R.close(out, want, R.turn_tolerance(want, size, dtype), "heads_first %s in_place %s pad %d" % (heads_first, in_place, pad))
        assert (dst[..., channels:] == 9.0).all()
        if not in_place:
            assert torch.equal(view, x)


def test_rotary_far_positions_and_back(odla, gpu_lib):
    """The largest and smallest int32 positions, frequencies above a turn per position; opposite frequencies turn back."""
    x = randn(gen(1), (1, 4, 2, 64), 0)
    pos = torch.tensor([[[2 ** 31 - 1, -2 ** 31, 0, 12345678]]], dtype=torch.int32, device="cuda")
    f = [7.3 * 1.7 ** (-i) for i in range(32)]
    d = odla.RotaryDesc(dtype=0, batch=1, tokens=4, heads=2, channels=64, x_batch=512, x_token=128, x_head=64, y_batch=512, y_token=128, y_head=64)
    y, back = torch.empty_like(x), torch.empty_like(x)
    there, home = odla.rotary_spec(f), odla.rotary_spec([-v for v in f])
    assert gpu_lib.b200_rotary(C.byref(there), C.byref(d), x.data_ptr(), y.data_ptr(), pos.data_ptr(), R.stream()) == 0
    assert gpu_lib.b200_rotary(C.byref(home), C.byref(d), y.data_ptr(), back.data_ptr(), pos.data_ptr(), R.stream()) == 0
    # the angle in exact whole numbers: the frequency as a fraction, times the position, modulo 2 pi to 40 digits
    from decimal import Decimal, getcontext
    getcontext().prec = 60
    two_pi = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494")
    ang = np.array([[float((Decimal(int(p)) * Decimal(v)) % two_pi) for v in f] for p in pos[0, 0].tolist()])
    c, s = (torch.tensor(fn(ang), device="cuda").unsqueeze(1) for fn in (np.cos, np.sin))
    a, b = x[0, ..., :32].double(), x[0, ..., 32:].double()
    want = torch.cat([a * c - b * s, a * s + b * c], -1)[None]
    size = (a.abs() + b.abs()).repeat(1, 1, 2)[None]
    R.close(y, want, R.turn_tolerance(want, size, 0))
    R.close(back, x.double(), 4 * R.turn_tolerance(x.double(), size, 0))     # two calls, each on a pair no longer than |a| + |b|


# ------------------------------------------------------------------------ append ----
@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("tokens,heads,kv,channels,pairs,page,interleaved", [(1, 12, 12, 64, 32, 16, True), (7, 8, 2, 128, 64, 24, False), (65, 4, 4, 96, 16, 1, False),
                                                                             (130, 0, 3, 64, 32, 100, True), (9, 5, 1, 13, 0, 7, False), (33, 6, 2, 24, 7, 8, True)])
def test_append(odla, gpu_lib, dtype, token_major, tokens, heads, kv, channels, pairs, page, interleaved):
    g = gen(dtype, tokens, channels)
    pages = -(-tokens // page) + 3
    row = randn(g, (tokens, heads + 2 * kv, channels), dtype)
    shape = (pages, page, kv, channels) if token_major else (pages, kv, page, channels)
    kc, vc = randn(g, shape, dtype), randn(g, shape, dtype)
    kv_view = [c.transpose(1, 2) if token_major else c for c in (kc, vc)]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    if tokens > 5:      # not kept: padding, and numbers that are no slots
        slots[1], slots[3], slots[4] = -1, pages * page, 1 << 40
    pos = torch.randint(0, 1 << 19, (1, tokens), generator=g, device="cuda", dtype=torch.int32)
    f = freqs(pairs)
    spec = odla.rotary_spec(f, interleaved=interleaved)
    want_rows, size = R.turned(row, pos, f, [0] * pairs, interleaved)
    want = [c.double().clone() for c in kv_view]
    tol = [torch.zeros_like(w) for w in want]
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            want[0][s // page, :, s % page] = want_rows[t, heads:heads + kv]
            tol[0][s // page, :, s % page] = R.turn_tolerance(want_rows, size, dtype)[t, heads:heads + kv]
            want[1][s // page, :, s % page] = row[t, heads + kv:].double()
    q_out = torch.full((tokens, max(heads, 1), channels), 9.0, dtype=row.dtype, device="cuda")
    cache = R.cache_of(odla, kv_view[0], dtype)
    st = row.stride(0)
    d = odla.AppendDesc(tokens=tokens, heads=heads, q_token=st, q_head=channels, k_token=st, k_head=channels, v_token=st, v_head=channels, y_token=q_out.stride(0), y_head=channels)
    at = [row.data_ptr() + row.element_size() * channels * n for n in (0, heads, heads + kv)]
    rc = gpu_lib.b200_paged_append(C.byref(cache), kc.data_ptr(), vc.data_ptr(), C.byref(d), C.byref(spec) if pairs else None, at[0] if heads else None, at[1], at[2],
                                   q_out.data_ptr() if heads else None, pos.data_ptr() if pairs else None, slots.data_ptr(), R.stream())
    assert rc == 0
    for got, w, t, what in zip(kv_view, want, tol, ("keys", "values")):
        R.close(got, w, t, what)
    if heads:
        R.close(q_out, want_rows[:, :heads], R.turn_tolerance(want_rows, size, dtype)[:, :heads], "queries")
    else:
        assert (q_out == 9.0).all()


# --------------------------------------------------------------------- attention ----
def attention_case(dtype, batch, queries, heads, kv, channels, page, prefix, lengths, token_major=False, spare=3, poison=True, seed=0, q_scale=2.0):
    g = gen(batch, queries, heads, channels, page, prefix, seed)
    width = max([-(-n // page) for n in lengths] + [1])
    shared = -(-prefix // page)
    used = shared + sum(-(-max(n, 0) // page) for n in lengths)
    pages = used + spare
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    shape = (pages, page, kv, channels) if token_major else (pages, kv, page, channels)
    caches = []
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    at = shared
    for i, n in enumerate(lengths):
        m = -(-max(n, 0) // page)
        table[i, :m] = order[at:at + m]
        at += m
    for _ in range(2):
        c = randn(g, shape, dtype)
        c = c.transpose(1, 2) if token_major else c
        if poison:      # every slot that no query sees holds NaN
            full = torch.full_like(c, float("nan"))
            for row, n in [(order[:shared], prefix)] + [(table[i], n) for i, n in enumerate(lengths)]:
                for j in range(-(-max(n, 0) // page)):
                    m = min(page, n - j * page)
                    full[int(row[j]), :, :m] = c[int(row[j]), :, :m]
            c = full
        caches.append(c)
    q = (q_scale * randn(g, (batch, queries, heads, channels), dtype).float()).to(R.TORCH[dtype])
    return q, caches[0], caches[1], order[:max(shared, 1)].contiguous(), table, torch.tensor(lengths, dtype=torch.int32, device="cuda")


def check_attention(odla, lib, case, prefix, scale=None, **kw):
    q, kc, vc, pp, table, lengths = case
    scale = R.scale_of(q.shape[-1]) if scale is None else scale
    want, tol = R.attention(q.cpu(), kc.cpu(), vc.cpu(), pp.cpu(), prefix, table.cpu(), lengths.cpu(), scale)
    y = R.call_attention(odla, lib, q, kc, vc, pp, prefix, table, lengths, scale, **kw)
    R.close(y, want, tol, "attention")
    return y


def test_attention_a_wait_that_runs_out_gives_nan_and_the_next_call_is_exact(odla, gpu_lib, monkeypatch):
    """The hook leaves one unit of the first block's ring unannounced; the products' wait for it ends after 256 attempts."""
    case = attention_case(1, 24, 1, 8, 2, 128, 16, 600, [30] * 24)
    monkeypatch.setenv("ODLA_B200_TEST_SKIP_STAGE", "1")
    monkeypatch.setenv("ODLA_B200_TEST_SPIN_LIMIT", "256")
    y = R.call_attention(odla, gpu_lib, *case[:4], 600, *case[4:], R.scale_of(128))
    torch.cuda.synchronize()
    assert torch.isnan(y).all()
    monkeypatch.delenv("ODLA_B200_TEST_SKIP_STAGE")
    monkeypatch.delenv("ODLA_B200_TEST_SPIN_LIMIT")
    check_attention(odla, gpu_lib, case, 600)


SHAPES = [  # batch, queries, heads, kv heads, channels, page, prefix, own lengths
    (1, 1, 1, 1, 64, 16, 0, [1]),
    (1, 1, 2, 1, 128, 16, 1, [0]),
    (3, 1, 12, 12, 64, 16, 200, [317, 5, 64]),
    (5, 1, 8, 2, 128, 24, 130, [0, 1, 127, 128, 129]),
    (4, 3, 8, 1, 128, 7, 33, [3, 2, 1, 50]),
    (2, 5, 28, 4, 128, 32, 300, [250, 77]),
    (1, 17, 4, 2, 64, 100, 0, [230]),
    (40, 1, 16, 2, 64, 8, 700, [(i * 13) % 90 for i in range(40)]),
    (6, 1, 32, 1, 128, 64, 513, [65, 0, 3, 200, 1, 64]),
    (9, 4, 8, 1, 128, 16, 1025, [4 + 11 * i for i in range(9)]),
    (33, 1, 8, 1, 64, 1, 260, [i % 5 for i in range(33)]),
    (34, 1, 8, 1, 128, 24, 1500, [i % 7 for i in range(34)]),
    (70, 2, 4, 1, 128, 16, 129, [2 + i % 9 for i in range(70)]),
    (24, 1, 6, 1, 64, 100, 2049, [0] * 24),
    (2, 9, 8, 1, 128, 24, 70, [400, 35]),
    (3, 20, 8, 1, 64, 16, 0, [300, 20, 7]),
    (1, 40, 8, 1, 128, 48, 200, [290]),
    (2, 70, 4, 1, 128, 7, 5, [200, 66]),
]


@pytest.mark.parametrize("dtype", [1, 2])
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(odla, gpu_lib, dtype, token_major, shape):
    check_attention(odla, gpu_lib, attention_case(dtype, *shape, token_major=token_major), shape[6])


@pytest.mark.parametrize("shape", [(3, 3, 12, 2, 64, 16, 0, [700, 33, 5]), (2, 8, 8, 1, 64, 24, 100, [1300, 40]), (5, 2, 20, 2, 128, 16, 0, [2, 1, 513, 128, 90]),
                                   (1, 8, 40, 8, 128, 100, 0, [2100]), (4, 4, 16, 1, 128, 7, 40, [0, 4, 31, 1025]), (40, 2, 24, 1, 64, 64, 0, [i * 29 % 300 for i in range(40)])])
def test_attention_teams_of_tiles(odla, gpu_lib, shape):
    """17 to 64 rows of a sequence: two or four tiles of 16, the last of them partly or wholly empty, over the same positions."""
    check_attention(odla, gpu_lib, attention_case(1, *shape), shape[6])
    check_attention(odla, gpu_lib, attention_case(2, *shape, token_major=True, seed=1), shape[6], scale=-0.1)


@pytest.mark.parametrize("queries,heads", [(3, 6), (5, 28)])
def test_attention_a_later_querys_infinity_in_teams(odla, gpu_lib, queries, heads):
    q, kc, vc, pp, table, lengths = attention_case(1, 2, queries, heads, heads // 6 if heads == 6 else 4, 64, 16, 0, [70, queries])
    for i, n in enumerate((70, queries)):
        vc[int(table[i, (n - 1) // 16]), :, (n - 1) % 16] = float("inf")      # only the last query sees it
    y = R.call_attention(odla, gpu_lib, q, kc, vc, None, 0, table, lengths, 0.125)
    assert torch.isfinite(y[:, :-1]).all() and not torch.isfinite(y[:, -1]).any()


def test_attention_sees_nothing(odla, gpu_lib):
    q, kc, vc, pp, table, lengths = attention_case(1, 4, 2, 4, 2, 64, 16, 0, [0, 1, 40, 0])
    lengths[3] = -5
    y = check_attention(odla, gpu_lib, (q, kc, vc, pp, table, lengths), 0)
    assert (y[0] == 0).all() and (y[1, 0] == 0).all() and (y[3] == 0).all() and y[1, 1].abs().max() > 0
    none = torch.zeros((4, 0), dtype=torch.int32, device="cuda")
    y = R.call_attention(odla, gpu_lib, q, kc, vc, None, 0, none, lengths, 0.125)
    assert (y == 0).all()


@pytest.mark.parametrize("prefix", [0, 90, 700])
def test_attention_bad_pages_are_not_seen(odla, gpu_lib, prefix):
    case = attention_case(2, 20, 1, 8, 1, 128, 16, prefix, [100] * 20)
    q, kc, vc, pp, table, lengths = case
    table[0, 2], table[1, :], table[2, 0], lengths[3] = -1, 1 << 30, kc.shape[0], 100000     # the last: longer than its table
    table[3, -1] = table[4, 0]
    kc.nan_to_num_(nan=0.5), vc.nan_to_num_(nan=0.5)      # (the last page's end is seen now)
    if prefix:
        pp[1] = -7
    check_attention(odla, gpu_lib, (q, kc, vc, pp, table, lengths), prefix)


def test_attention_a_later_querys_infinity_stays_its_own(odla, gpu_lib):
    q, kc, vc, pp, table, lengths = attention_case(1, 2, 3, 4, 2, 64, 16, 20, [37, 3])
    for i, n in enumerate((37, 3)):
        vc[int(table[i, (n - 1) // 16]), :, (n - 1) % 16] = float("inf")      # only the last query sees it
    y = R.call_attention(odla, gpu_lib, q, kc, vc, pp, 20, table, lengths, 0.125)
    assert torch.isfinite(y[:, :2]).all() and not torch.isfinite(y[:, 2]).any()
    clean = vc.clone()
    clean[torch.isinf(clean)] = 0.25
    want, tol = R.attention(q.cpu(), kc.cpu(), clean.cpu(), pp.cpu(), 20, table.cpu(), lengths.cpu(), 0.125)
    R.close(y[:, :2], want[:, :2], tol[:, :2])


@pytest.mark.parametrize("prefix", [0, 600])
def test_attention_extreme_scores(odla, gpu_lib, prefix):
    """One position outweighs all others by hundreds of units, wherever it lies; scores far below zero everywhere else."""
    case = attention_case(2, 24, 1, 4, 1, 64, 16, prefix, [70] * 24, q_scale=12.0)
    q, kc, vc, pp, table, lengths = case
    kc[int(table[0, 4]), 0, 1] = q[0, 0, 0] * 3
    if prefix:
        kc[int(pp[30]), 0, 5] = q[7, 0, 1] * 3
    check_attention(odla, gpu_lib, case, prefix)
    check_attention(odla, gpu_lib, case, prefix, scale=0.0)
    check_attention(odla, gpu_lib, case, prefix, scale=-0.2)


@pytest.mark.parametrize("dtype", [1, 2])
@pytest.mark.parametrize("prefix,batch,channels", [(0, 3, 64), (600, 24, 128), (600, 80, 64)])
def test_attention_scores_of_minus_infinity_weigh_nothing(odla, gpu_lib, dtype, prefix, batch, channels):
    """All scores minus infinity: zeros.  All but one: that position's value, to the rounding of one weight over itself."""
    case = attention_case(dtype, batch, 1, 4, 1, channels, 16, prefix, [70] * batch, poison=False)
    q, kc, vc, pp, table, lengths = case
    q[..., 0] = 1.0
    kc[..., 0] = float("-inf")
    y = R.call_attention(odla, gpu_lib, q, kc, vc, pp, prefix, table, lengths, 0.125)
    assert (y == 0).all()
    if prefix:
        kc[int(pp[20]), 0, 7, 0] = 0.0
        want = vc[int(pp[20]), 0, 7].expand(batch, 4, channels)
    else:
        want = torch.zeros((batch, 4, channels), dtype=q.dtype, device="cuda")
        for b in range(batch):
            kc[int(table[b, 2]), 0, 3, 0] = 0.0
            want[b] = vc[int(table[b, 2]), 0, 3]
    y = R.call_attention(odla, gpu_lib, q, kc, vc, pp, prefix, table, lengths, 0.125)
    # (w v) / w: two roundings in 32 bits, which may move a value of the type by a step only where they cross its rounding border; v itself is no border
    assert torch.equal(y[:, 0], want)


def test_attention_strides_and_neighbours(odla, gpu_lib):
    """Queries inside a projection's rows, results inside a wider buffer: what lies between stays as it was."""
    q, kc, vc, pp, table, lengths = attention_case(1, 3, 2, 6, 2, 64, 16, 50, [33, 64, 2])
    wide = torch.full((3, 2, 10, 80), 5.0, dtype=q.dtype, device="cuda")
    wide[:, :, 2:8, 8:72] = q
    out = torch.full((5, 2, 9, 72), 6.0, dtype=q.dtype, device="cuda")
    y = out[1:4, :, 1:7, :64]
    want, tol = R.attention(q.cpu(), kc.cpu(), vc.cpu(), pp.cpu(), 50, table.cpu(), lengths.cpu(), 0.125)
    R.call_attention(odla, gpu_lib, wide[:, :, 2:8, 8:72], kc, vc, pp, 50, table, lengths, 0.125, y=y)
    R.close(y, want, tol)
    out[1:4, :, 1:7, :64] = 6.0
    assert (out == 6.0).all()


def test_attention_replays_follow_their_lengths(odla, gpu_lib):
    """A captured call reads lengths, tables and queries when it runs; runs of the same inputs have the same bits."""
    q, kc, vc, pp, table, lengths = attention_case(2, 20, 1, 8, 2, 128, 16, 400, [90] * 20)
    y = torch.empty_like(q)
    R.call_attention(odla, gpu_lib, q, kc, vc, pp, 400, table, lengths, 0.088, y=y)
    first = y.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    ws = torch.empty(1 << 26, dtype=torch.uint8, device="cuda")
    with torch.cuda.graph(graph, stream=side):
        R.call_attention(odla, gpu_lib, q, kc, vc, pp, 400, table, lengths, 0.088, y=y, workspace=ws)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, first)
    lengths.copy_(torch.arange(20, device="cuda") * 4 + 1)
    q.mul_(0.5)
    graph.replay()
    want, tol = R.attention(q.cpu(), kc.cpu(), vc.cpu(), pp.cpu(), 400, table.cpu(), lengths.cpu(), 0.088)
    R.close(y, want, tol)


# ---------------------------------------------------------------------- sampling ----
def params(g, rows):
    def pick(values, dtype=torch.float32):
        return torch.tensor(values, dtype=dtype, device="cuda")[torch.randint(0, len(values), (rows,), generator=g, device="cuda")]
    return pick([0.0, 0.3, 0.7, 1.0, 1.0, 2.5]), pick([0, -1, 1, 2, 17, 50, 400], torch.int32), pick([1.0, 1.5, 0.0, 0.5, 0.9, 0.99]), pick([0.0, 0.0, 0.05, 0.3, 1.0, 2.0])


def check_sample(odla, lib, logits, p, u, dtype):
    got = R.call_sample(odla, lib, logits, *p, u, dtype).cpu().numpy()
    want = R.sample(logits.double().cpu().numpy(), *[None if x is None else x.cpu().numpy() for x in p], u.cpu().numpy())
    assert (got == want).all(), np.flatnonzero(got != want)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("rows,vocab,pad", [(1, 1, 0), (9, 2, 0), (40, 31, 1), (40, 511, 0), (40, 513, 3), (60, 1000, 0), (30, 8193, 8), (3, 30522, 0), (20, 30522, 0), (200, 5000, 0),
                                           (5, 131072, 0), (2, 262144, 0)])
def test_sample(odla, gpu_lib, dtype, rows, vocab, pad):
    g = gen(dtype, rows, vocab)
    wide = (3 * torch.randn((rows, vocab + pad), generator=g, device="cuda")).to(R.TORCH[dtype])
    logits = wide[:, :vocab]
    u = torch.rand(rows, generator=g, device="cuda")
    u[::7] = 0.0
    u[3::7] = 1.0 - 2.0 ** -24
    check_sample(odla, gpu_lib, logits, params(g, rows), u, dtype)
    check_sample(odla, gpu_lib, logits, (None, None, None, None), u, dtype)


@pytest.mark.parametrize("dtype", [0, 2])
@pytest.mark.parametrize("spread", [0.05, 1.0, 20.0])
@pytest.mark.parametrize("rows,vocab", [(64, 3000), (24, 50001), (150, 32000)])
def test_sample_each_filter_alone_and_together(odla, gpu_lib, dtype, spread, rows, vocab):
    """Flat, ordinary and steep rows; top-k on both sides of 1024, top-p from nearly nothing to nearly all."""
    g = gen(rows, vocab, int(spread * 100), dtype)
    logits = (spread * torch.randn((rows, vocab), generator=g, device="cuda")).to(R.TORCH[dtype])
    u = torch.rand(rows, generator=g, device="cuda")

    def pick(values, dtype=torch.float32):
        return torch.tensor(values, dtype=dtype, device="cuda")[torch.randint(0, len(values), (rows,), generator=g, device="cuda")]
    T, k, p, m = pick([0.2, 0.7, 1.0, 1.7]), pick([1, 3, 40, 1000, 1024, 1025, 2000, 10 ** 6], torch.int32), pick([0.01, 0.3, 0.8, 0.95, 0.999, 0.999999]), pick([1e-6, 0.01, 0.2, 0.9])
    for params in ((T, None, None, None), (T, k, None, None), (T, None, p, None), (T, None, None, m), (T, None, p, m), (T, k, p, None), (T, k, p, m)):
        check_sample(odla, gpu_lib, logits, params, u, dtype)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("vocab", [100, 4096, 40000])
def test_sample_ties(odla, gpu_lib, dtype, vocab):
    """Few distinct logits: the cuts of top-k and top-p fall between equal ones; -0 and +0 are equal."""
    g = gen(dtype, vocab, 5)
    rows = 48
    logits = torch.randint(-2, 3, (rows, vocab), generator=g, device="cuda").float() / 2
    logits[::3] = 0.0
    logits[1::6] = torch.where(torch.rand((1, vocab), generator=g, device="cuda") < 0.5, -0.0, 0.0)
    t, k, p, m = params(g, rows)
    k = torch.randint(0, vocab + 2, (rows,), generator=g, device="cuda", dtype=torch.int32)
    # (top_p of an eighth's multiple, and temperatures that are powers of two: a border on a tie is the same border in both)
    p = torch.randint(1, 9, (rows,), generator=g, device="cuda").float() / 8
    u = torch.rand(rows, generator=g, device="cuda")
    check_sample(odla, gpu_lib, logits.to(R.TORCH[dtype]), (t, k, p, m), u, dtype)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("vocab", [50, 9000])
def test_sample_masks_infinities_and_nan(odla, gpu_lib, dtype, vocab):
    g = gen(dtype, vocab, 6)
    x = 2 * torch.randn((14, vocab), generator=g, device="cuda")
    inf = float("inf")
    x[0] = -inf
    x[1] = float("nan")
    x[2, 1:] = -inf
    x[3, :-1] = -inf
    x[4, ::2] = float("nan")
    x[5, 7] = inf
    x[6, 7::5] = inf
    x[7] = inf
    x[8] = torch.finfo(R.TORCH[dtype]).min
    x[9, 3:] = torch.finfo(R.TORCH[dtype]).min
    x[10, :40] = float("nan")
    x[11, 20:] = -inf
    x[12] = torch.finfo(R.TORCH[dtype]).max
    x[13, 5] = torch.finfo(R.TORCH[dtype]).max
    u = torch.full((14,), 0.4, device="cuda")
    x = x.to(R.TORCH[dtype])
    for T, k, p, m in ((1.0, 0, 1.0, 0.0), (0.5, 5, 0.9, 0.01), (0.0, 0, 1.0, 0.0), (2.0, 30, 0.3, 0.0), (1e-30, 0, 0.99, 0.0), (1e30, 0, 0.5, 0.2)):
        check_sample(odla, gpu_lib, x, tuple(torch.full((14,), v, device="cuda", dtype=torch.int32 if i == 1 else torch.float32) for i, v in enumerate((T, k, p, m))), u, dtype)


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_sample_masks_that_leave_parts_of_a_row(odla, gpu_lib, dtype):
    """Whole stretches of a long row allow nothing, or less than k; the largest logits lie all in one place, or in order."""
    g = gen(77, dtype)
    rows, vocab = 40, 90000
    x = 2 * torch.randn((rows, vocab), generator=g, device="cuda")
    inf = float("inf")
    x[0:4, 20000:] = -inf
    x[4:8, :85000] = -inf
    x[8:12, 17:] = -inf
    x[12:16] = x[12:16].sort(dim=-1, descending=True).values
    x[16:20] = x[16:20].sort(dim=-1).values
    x[20:24, 30000:30500] += 30
    x[24:28, ::3] = float("nan")
    x[28:32] = -inf
    x[28:30, 89999] = 1.0
    x[32:34, 70000] = inf
    x[34:36, 5] = torch.finfo(R.TORCH[dtype]).min
    x[36:38] = x[36:38].round()
    u = torch.rand(rows, generator=g, device="cuda")
    x = x.to(R.TORCH[dtype])
    for k, p in ((3, 1.0), (40, 0.9), (300, 0.99), (1000, 0.5), (0, 0.8)):
        check_sample(odla, gpu_lib, x, (torch.full((rows,), 0.9, device="cuda"), torch.full((rows,), k, dtype=torch.int32, device="cuda"), torch.full((rows,), p, device="cuda"), None), u, dtype)


def test_sample_leaves_the_rest_and_strides(odla, gpu_lib):
    g = gen(8)
    logits = torch.randn((4, 700), generator=g, device="cuda")
    out = torch.full((9,), -3, dtype=torch.int32, device="cuda")
    u = torch.rand(4, generator=g, device="cuda")
    R.call_sample(odla, gpu_lib, logits, None, None, None, None, u, 0, tokens=out[2:6])
    assert (out[:2] == -3).all() and (out[6:] == -3).all() and (out[2:6] >= 0).all()
    same = R.call_sample(odla, gpu_lib, logits[:1].expand(4, 700), None, None, None, None, u, 0, row=0)
    assert (same.cpu().numpy() == R.sample(logits[:1].expand(4, 700).double().cpu().numpy(), None, None, None, None, u.cpu().numpy())).all()


# ------------------------------------------------------------ far offsets, replays ----
def test_offsets_beyond_32_bits(odla, gpu_lib):
    """Pages, tokens and rows more than 2^32 elements apart (16 GB of which a few rows are touched)."""
    g = gen(64)
    far = (1 << 32) + 64
    big = torch.empty(2 * far + 4096, dtype=torch.float16, device="cuda")
    kc = torch.as_strided(big, (2, 1, 16, 64), (far, 1024, 64, 1))
    vc = torch.as_strided(big, (2, 1, 16, 64), (far, 1024, 64, 1), 2048)
    kc.copy_(randn(g, (2, 1, 16, 64), 1)), vc.copy_(randn(g, (2, 1, 16, 64), 1))
    # append to the far page
    row = randn(g, (2, 3, 64), 1)
    slots = torch.tensor([16 + 15, 16 + 14], device="cuda")
    pos = torch.tensor([[3, 4]], dtype=torch.int32, device="cuda")
    f = freqs(32)
    spec, cache = odla.rotary_spec(f), R.cache_of(odla, kc, 1)
    out = torch.empty((2, 1, 64), dtype=torch.float16, device="cuda")
    d = odla.AppendDesc(tokens=2, heads=1, q_token=192, q_head=64, k_token=192, k_head=64, v_token=192, v_head=64, y_token=64, y_head=64)
    assert gpu_lib.b200_paged_append(C.byref(cache), kc.data_ptr(), vc.data_ptr(), C.byref(d), C.byref(spec), row.data_ptr(), row.data_ptr() + 128, row.data_ptr() + 256, out.data_ptr(),
                                     pos.data_ptr(), slots.data_ptr(), R.stream()) == 0
    want, size = R.turned(row, pos, f, [0] * 32, False)
    R.close(kc[1, 0, [15, 14]], want[:, 1], R.turn_tolerance(want, size, 1)[:, 1])
    assert torch.equal(vc[1, 0, [15, 14]], row[:, 2])
    # attention over both pages, by small tiles and by wide ones
    for batch in (1, 20):
        q = randn(g, (batch, 1, 1, 64), 1)
        table = torch.tensor([[1, 0]] * batch, dtype=torch.int32, device="cuda")
        pages = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
        check_attention(odla, gpu_lib, (q, kc, vc, pages, table, torch.full((batch,), 20, dtype=torch.int32, device="cuda")), 32)
    # rotary and sampling from rows far apart
    x = torch.as_strided(big, (1, 2, 1, 64), (0, far, 64, 1), 8192 - 4096)
    x.copy_(randn(g, (1, 2, 1, 64), 1))
    y = torch.empty((1, 2, 1, 64), dtype=torch.float16, device="cuda")
    p = torch.tensor([[[5, 6]]], dtype=torch.int32, device="cuda")
    rd = odla.RotaryDesc(dtype=1, batch=1, tokens=2, heads=1, channels=64, x_batch=0, x_token=far, x_head=64, y_batch=0, y_token=64, y_head=64)
    assert gpu_lib.b200_rotary(C.byref(spec), C.byref(rd), x.data_ptr(), y.data_ptr(), p.data_ptr(), R.stream()) == 0
    want, size = R.turned(x, p, f, [0] * 32, False)
    R.close(y, want, R.turn_tolerance(want, size, 1))
    logits = torch.as_strided(big, (2, 1000), (far, 1))
    logits.copy_(randn(g, (2, 1000), 1))
    u = torch.tensor([0.3, 0.8], device="cuda")
    check_sample(odla, gpu_lib, logits, (None, None, None, None), u, 1)


def captured(call):
    """`call` as a graph on a stream of its own."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call()
    return graph


def test_captured_rotary_append_and_sample_follow_their_inputs(odla, gpu_lib):
    g = gen(65)
    x, y = randn(g, (1, 9, 4, 64), 2), torch.empty((1, 9, 4, 64), dtype=torch.bfloat16, device="cuda")
    pos = torch.arange(9, dtype=torch.int32, device="cuda").view(1, 1, 9)
    f = freqs(32)
    spec = odla.rotary_spec(f)
    rd = odla.RotaryDesc(dtype=2, batch=1, tokens=9, heads=4, channels=64, x_batch=2304, x_token=256, x_head=64, y_batch=2304, y_token=256, y_head=64)
    kc, vc = (torch.zeros((4, 2, 8, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cache = R.cache_of(odla, kc, 2)
    ad = odla.AppendDesc(tokens=9, heads=0, k_token=256, k_head=64, v_token=256, v_head=64)
    slots = torch.arange(9, device="cuda")
    logits, u = randn(g, (5, 3000), 2), torch.rand(5, generator=g, device="cuda")
    k = torch.full((5,), 40, dtype=torch.int32, device="cuda")
    tokens = torch.empty(5, dtype=torch.int32, device="cuda")

    def calls():
        assert gpu_lib.b200_rotary(C.byref(spec), C.byref(rd), x.data_ptr(), y.data_ptr(), pos.data_ptr(), R.stream()) == 0
        assert gpu_lib.b200_paged_append(C.byref(cache), kc.data_ptr(), vc.data_ptr(), C.byref(ad), None, None, y.data_ptr(), y.data_ptr() + 256, None, None, slots.data_ptr(),
                                         R.stream()) == 0
        R.call_sample(odla, gpu_lib, logits, None, k, None, None, u, 2, tokens=tokens)
    calls()
    graph = captured(calls)
    spec.frequency[0] = 77.0                 # descriptors are read during the call, not when the graph runs
    rd.tokens, ad.tokens = 1, 0
    for i in range(3):
        x.copy_(randn(g, tuple(x.shape), 2)), pos.add_(1000), slots.add_(3), logits.copy_(randn(g, (5, 3000), 2)), u.copy_(torch.rand(5, generator=g, device="cuda"))
        graph.replay()
        want, size = R.turned(x, pos, f, [0] * 32, False)
        R.close(y, want, R.turn_tolerance(want, size, 2))
        at = slots.tolist()
        assert torch.equal(kc.transpose(1, 2).reshape(32, 2, 64)[at], y[0, :, :2]) and torch.equal(vc.transpose(1, 2).reshape(32, 2, 64)[at], y[0, :, 2:])
        assert (tokens.cpu().numpy() == R.sample(logits.double().cpu().numpy(), None, k.cpu().numpy(), None, None, u.cpu().numpy())).all()


def test_calls_on_two_streams_at_once(odla, gpu_lib):
    cases = [attention_case(2, 24, 1, 8, 2, 128, 16, 500 + 100 * i, [80] * 24, seed=i) for i in range(2)]
    logits = [3 * randn(gen(70 + i), (30, 20000), 0) for i in range(2)]
    us = [torch.rand(30, generator=gen(80 + i), device="cuda") for i in range(2)]
    alone = [R.call_attention(odla, gpu_lib, *c[:4], 500 + 100 * i, *c[4:], 0.088) for i, c in enumerate(cases)]
    tokens = [R.call_sample(odla, gpu_lib, l, None, None, None, None, u, 0) for l, u in zip(logits, us)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((R.call_attention(odla, gpu_lib, *cases[i][:4], 500 + 100 * i, *cases[i][4:], 0.088),
                               R.call_sample(odla, gpu_lib, logits[i], None, None, None, None, us[i], 0)))
    torch.cuda.synchronize()
    for i in range(2):
        for y, t in got[i]:
            assert torch.equal(y, alone[i]) and torch.equal(t, tokens[i])


# --------------------------------------------------------------------- a whole step ----
def test_a_decoding_loop_next_to_planned_graphs(odla, gpu_lib):
    """What a program does for each new token: the projection as a planned graph, append, attention, the output layer as a planned
    graph, sampling.  Every stage against its 64-bit form on what it was given; three sequences behind one prompt, one slot of the batch unused."""
    g = gen(90)
    B, H, KH, D, V, PS, P, steps = 4, 4, 2, 64, 700, 8, 21, 6
    hidden, width = H * D, (H + 2 * KH) * D
    rng = np.random.default_rng(3)
    w_in, w_out = ((rng.standard_normal((hidden, n)) / np.sqrt(hidden)).astype(np.float32) for n in (width, V))
    table_emb = randn(g, (V, hidden), 1)
    project, answer = odla.Graph(gpu_lib, "project", fp16=True, n_gpus=1), None
    project.Output(project.Gemm(project.Argument("x", (B, hidden), odla.FLOAT16), False, project.Constant("w", w_in), False, 1.0, 0.0, None, (B, width), "qkv"))
    project.context()
    answer = odla.Graph(gpu_lib, "answer", fp16=True, n_gpus=1)
    answer.Output(answer.Gemm(answer.Argument("c", (B, hidden), odla.FLOAT16), False, answer.Constant("w", w_out), False, 1.0, 0.0, None, (B, V), "logits"))
    answer.context()
    pages = 16
    kc, vc = (randn(g, (pages, KH, PS, D), 1) for _ in range(2))
    prefix_pages = torch.tensor([5, 2, 9], dtype=torch.int32, device="cuda")
    table = torch.tensor([[0], [1], [3], [-1]], dtype=torch.int32, device="cuda")
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    x = randn(g, (B, hidden), 1)
    qkv, turned, ctx = (torch.empty((B, n), dtype=torch.float16, device="cuda") for n in (width, hidden, hidden))
    logits, tokens = torch.empty((B, V), dtype=torch.float16, device="cuda"), torch.empty(B, dtype=torch.int32, device="cuda")
    f = freqs(D // 2)
    spec, cache = odla.rotary_spec(f), R.cache_of(odla, kc, 1)
    ad = odla.AppendDesc(tokens=B, heads=H, q_token=width, q_head=D, k_token=width, k_head=D, v_token=width, v_head=D, y_token=hidden, y_head=D)
    for step in range(steps):
        torch.cuda.synchronize()
        project.bind_input("x", x.data_ptr()), project.bind_output("qkv", qkv.data_ptr())
        assert project.execute() == odla.SUCCESS
        want = x.double() @ torch.tensor(w_in, device="cuda").half().double()
        # 256 products summed in fp32, rounded once
        bound = x.double().abs() @ torch.tensor(w_in, device="cuda").half().double().abs()
        R.close(qkv, want, bound * 260 * 2.0 ** -24 + want.abs() * 2.0 ** -11 + 2.0 ** -25, "projection")
        positions = torch.full((1, B), P + step, dtype=torch.int32, device="cuda")
        slots = torch.where(table[:, 0] >= 0, table[:, 0].long() * PS + step, -1)
        lengths.copy_(torch.where(table[:, 0] >= 0, step + 1, 0))
        es = 2 * D
        assert gpu_lib.b200_paged_append(C.byref(cache), kc.data_ptr(), vc.data_ptr(), C.byref(ad), C.byref(spec), qkv.data_ptr(), qkv.data_ptr() + H * es, qkv.data_ptr() + (H + KH) * es,
                                         turned.data_ptr(), positions.data_ptr(), slots.data_ptr(), R.stream()) == 0
        rows, size = R.turned(qkv.view(B, H + 2 * KH, D), positions, f, [0] * (D // 2), False)
        tol = R.turn_tolerance(rows, size, 1)
        R.close(turned.view(B, H, D), rows[:, :H], tol[:, :H], "queries")
        for b in range(3):
            R.close(kc[int(table[b, 0]), :, step], rows[b, H:H + KH], tol[b, H:H + KH], "keys")
            assert torch.equal(vc[int(table[b, 0]), :, step], qkv.view(B, -1, D)[b, H + KH:])
        y = R.call_attention(odla, gpu_lib, turned.view(B, 1, H, D), kc, vc, prefix_pages, P, table, lengths, 0.125, y=ctx.view(B, 1, H, D))
        want, tol = R.attention(turned.view(B, 1, H, D).cpu(), kc.cpu(), vc.cpu(), prefix_pages.cpu(), P, table.cpu(), lengths.cpu(), 0.125)
        R.close(y, want, tol, "attention")
        torch.cuda.synchronize()
        answer.bind_input("c", ctx.data_ptr()), answer.bind_output("logits", logits.data_ptr())
        assert answer.execute() == odla.SUCCESS
        T, k, p = torch.tensor([0.7, 1.0, 0.0, 1.0], device="cuda"), torch.tensor([0, 30, 0, 0], dtype=torch.int32, device="cuda"), torch.tensor([0.9, 1.0, 1.0, 0.5], device="cuda")
        u = torch.rand(B, generator=g, device="cuda")
        R.call_sample(odla, gpu_lib, logits, T, k, p, None, u, 1, tokens=tokens)
        assert (tokens.cpu().numpy() == R.sample(logits.double().cpu().numpy(), T.cpu().numpy(), k.cpu().numpy(), p.cpu().numpy(), None, u.cpu().numpy())).all()
        x.copy_(table_emb[tokens.long()])
    project.close()
    answer.close()
