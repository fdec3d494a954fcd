"""The norm, attention of a chunk and log probabilities through the C ABI against plain 64-bit forms."""
import ctypes as C

import pytest
import torch

import decode_ref as R
import prompt_ref as P

pytestmark = pytest.mark.gpu
INF = float("inf")


def gen(*seed):
    return torch.Generator(device="cuda").manual_seed(sum(int(s) * 1009 ** i for i, s in enumerate(seed)) % (1 << 31))


def randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(R.TORCH[dtype])


def captured(call):
    """The call in a CUDA graph, on a stream of its own."""
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        call()
    return graph


# -------------------------------------------------------------------------- norm ----
def check_norm(odla, lib, dtype, rows, heads, channels, quant=0, group=0, residual=True, weight=0, pad=0, with_y=True, offset=0.0, in_place=False, seed=0, given=0.02):
    g = gen(dtype, rows, channels, quant, group, seed)
    wide = [torch.full((rows, heads + 1, channels + pad), 9.0, dtype=R.TORCH[dtype], device="cuda") for _ in range(4)]
    x, r, s, y = (t[:, :heads, :channels] for t in wide)
    x.copy_(randn(g, x.shape, dtype))
    x[..., channels // 3] *= 30
    r.copy_(randn(g, x.shape, dtype) * 2)
    w = None if weight is None else (1 + 0.3 * torch.randn(channels, generator=g, device="cuda")).to(R.TORCH[weight])
    if not residual:
        r = s = None
    q8 = scales = None
    if quant:
        q_wide = torch.full((rows, heads + 1, channels + pad), 33, dtype=torch.uint8, device="cuda")
        q8 = q_wide[:, :heads, :channels]
        scales = torch.full((rows, heads, channels // group), 7.0, device="cuda") if group else torch.full((1,), given, device="cuda")
    h, want = P.norm(x, r, w, 1e-5, offset)
    if in_place:
        s, y = (r, x) if residual else (None, x)
    if not with_y:
        y = None
    assert P.call_norm(odla, lib, x, r, w, s, y, q8, scales, quant, group, 1e-5, offset) == 0
    if s is not None:
        assert torch.equal(s, h)
    if y is not None:
        P.near(y, want, P.norm_tolerance(want, dtype), "y")
    if quant:
        if group:
            top = want.unflatten(-1, (-1, group)).abs().amax(-1) / P.MOST[quant]
            P.near(scales, top, top * (P.NORM + 2 * P.U), "scales")
        values, tol = P.eight_bits(want, quant, scales, not group)
        got = q8.view(torch.int8 if quant == 1 else torch.float8_e4m3fn).double()
        sc = scales.double().repeat_interleave(channels // max(scales.shape[-1], 1), -1) if group else scales.double()
        P.near(got * sc, values, tol, "8 bits")
        q_wide[:, :heads, :channels] = 33
        assert (q_wide == 33).all()
    for t in wide:
        t[:, :heads, :channels] = 9.0
        assert (t == 9.0).all()


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("rows,heads,channels", [(1, 1, 1), (1, 1, 768), (3, 1, 7), (5, 1, 1001), (64, 1, 4096), (2, 1, 32768), (2, 1, 32761), (37, 12, 64), (9, 5, 128), (300, 3, 96), (4, 2, 8), (3, 1, 16384),
                                                 (7, 1, 5120), (2, 3, 250), (1, 1, 8200), (0, 1, 64)])
def test_norm(odla, gpu_lib, dtype, rows, heads, channels):
    check_norm(odla, gpu_lib, dtype, rows, heads, channels, weight=0)
    check_norm(odla, gpu_lib, dtype, rows, heads, channels, residual=False, weight=None, offset=0.5)
    check_norm(odla, gpu_lib, dtype, rows, heads, channels, weight=dtype, pad=8, offset=1.0)
    check_norm(odla, gpu_lib, dtype, rows, heads, channels, weight=2, pad=3)
    check_norm(odla, gpu_lib, dtype, rows, heads, channels, weight=1, in_place=True, pad=8)
    check_norm(odla, gpu_lib, dtype, rows, heads, channels, weight=0, residual=False, in_place=True)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("quant", [1, 2])
@pytest.mark.parametrize("rows,heads,channels,group", [(1, 1, 768, 768), (5, 1, 5120, 128), (3, 1, 4096, 4096), (64, 1, 4096, 32), (9, 5, 128, 128), (9, 5, 128, 32), (4, 3, 96, 24), (2, 1, 1001, 1001), (6, 1, 8, 8),
                                                       (3, 1, 32768, 8), (2, 1, 32768, 32768), (2, 1, 4608, 1536), (11, 2, 64, 0), (3, 1, 5120, 0), (2, 1, 333, 0), (3, 1, 7, 7), (4, 1, 1000, 40)])
def test_norm_in_8_bits(odla, gpu_lib, dtype, quant, rows, heads, channels, group):
    check_norm(odla, gpu_lib, dtype, rows, heads, channels, quant, group)
    check_norm(odla, gpu_lib, dtype, rows, heads, channels, quant, group, residual=False, with_y=False, weight=dtype, pad=8)
    check_norm(odla, gpu_lib, dtype, rows, heads, channels, quant, group, weight=None, pad=1, in_place=True)


@pytest.mark.parametrize("quant", [0, 1, 2])
def test_norm_of_the_sum_alone_and_of_zeros(odla, gpu_lib, quant):
    x = torch.zeros((4, 1, 256), dtype=torch.bfloat16, device="cuda")
    x[1] = 1.0
    x[2, 0, 64:] = 1.0
    r, s = torch.ones_like(x), torch.empty_like(x)
    assert P.call_norm(odla, gpu_lib, x, r, None, total=s) == 0
    assert torch.equal(s, x + r)
    y = torch.full_like(x, 7.0)
    q = torch.full((4, 1, 256), 55, dtype=torch.uint8, device="cuda") if quant else None
    scales = torch.full((4, 1, 4), 7.0, device="cuda")
    assert P.call_norm(odla, gpu_lib, x, y=y, quantised=q, scales=scales if quant else None, quant=quant, group=64 if quant else 0, epsilon=0.0) == 0
    # 0 / sqrt(0 + 0) is not a number, as the formula says; with an epsilon it is zero
    assert y[0].isnan().all() and (y[1] == 1).all()
    assert P.call_norm(odla, gpu_lib, x, y=y, quantised=q, scales=scales if quant else None, quant=quant, group=64 if quant else 0, epsilon=1e-6) == 0
    assert (y[0] == 0).all() and (y[2, 0, :64] == 0).all()
    if quant:
        assert (q[0] == 0).all() and (scales[0] == 0).all() and (q[2, 0, :64] == 0).all() and scales[2, 0, 0] == 0 and (scales[2, 0, 1:] > 0).all()


@pytest.mark.parametrize("quant", [1, 2])
@pytest.mark.parametrize("group", [64, 256])
def test_norm_scales_tell_of_infinities(odla, gpu_lib, quant, group):
    x = torch.ones((3, 1, 256), device="cuda")
    x[0, 0, 5], x[1, 0, 70] = INF, float("nan")
    w = torch.ones(256, device="cuda")
    q, scales = torch.empty((3, 1, 256), dtype=torch.uint8, device="cuda"), torch.empty((3, 1, 256 // group), device="cuda")
    y = torch.empty_like(x)
    assert P.call_norm(odla, gpu_lib, x, weight=w, y=y, quantised=q, scales=scales, quant=quant, group=group) == 0
    want = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    assert torch.equal(y.isnan(), want.isnan())
    bad = want.unflatten(-1, (-1, group)).isnan().any(-1)
    assert not scales[bad].isfinite().any() and scales[~bad].isfinite().all()


def test_norm_replays_and_other_streams(odla, gpu_lib):
    """A captured call follows its buffers; two calls on two streams at once give what each gives alone."""
    g = gen(3)
    x, r, w = randn(g, (65, 1, 2048), 2), randn(g, (65, 1, 2048), 2), randn(g, (2048,), 0)
    s, y = torch.empty_like(x), torch.empty_like(x)
    q, scales = torch.empty(x.shape, dtype=torch.uint8, device="cuda"), torch.empty((65, 1, 16), device="cuda")

    def call():
        assert P.call_norm(odla, gpu_lib, x, r, w, s, y, q, scales, 2, 128) == 0
    graph = captured(call)
    for scale in (1.0, 0.3):
        x.mul_(scale)
        graph.replay()
        h, want = P.norm(x, r, w, 1e-6, 0.0)
        assert torch.equal(s, h)
        P.near(y, want, P.norm_tolerance(want, 2))
        first = [t.clone() for t in (s, y, q, scales)]
        call()
        assert all(torch.equal(a, b) for a, b in zip(first, (s, y, q, scales)))
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(x) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, out in zip(streams, outs):
            with torch.cuda.stream(st):
                assert P.call_norm(odla, gpu_lib, s, weight=w, y=out) == 0
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1])


def test_norm_far_rows(odla, gpu_lib):
    """Rows whose offsets pass 32 bits."""
    step = (1 << 31) + 64
    big = torch.empty(2 * step + 256, dtype=torch.float16, device="cuda")
    x = torch.as_strided(big, (3, 1, 128), (step, 128, 1))
    x.copy_(randn(gen(5), (3, 1, 128), 1))
    _, want = P.norm(x, None, None, 1e-6, 0.0)
    assert P.call_norm(odla, gpu_lib, x, y=x) == 0
    P.near(x, want, P.norm_tolerance(want, 1))


# ------------------------------------------------------------------------- chunk ----
def chunk_case(dtype, new, lengths, heads, kv, channels, page, prefix, token_major=False, spare=3, poison=True, seed=0, q_scale=2.0, behind=5):
    g = gen(dtype, len(new), sum(new), heads, channels, page, prefix, seed)
    width = max([-(-n // page) for n in lengths] + [1])
    shared = -(-prefix // page)
    used = shared + sum(-(-max(n, 0) // page) for n in lengths)
    pages = used + spare
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(new), width), -1, dtype=torch.int32, device="cuda")
    at = shared
    for i, n in enumerate(lengths):
        m = -(-max(n, 0) // page)
        table[i, :m] = order[at:at + m]
        at += m
    caches = []
    for _ in range(2):
        c = randn(g, (pages, page, kv, channels) if token_major else (pages, kv, page, channels), dtype)
        c = c.transpose(1, 2) if token_major else c
        if poison:      # every slot that no sequence has a position in holds NaN
            full = torch.full_like(c, float("nan"))
            for row, n in [(order[:shared], prefix)] + [(table[i], n) for i, n in enumerate(lengths)]:
                for j in range(-(-max(n, 0) // page)):
                    m = min(page, n - j * page)
                    full[int(row[j]), :, :m] = c[int(row[j]), :, :m]
            c = full
        caches.append(c)
    q = (q_scale * randn(g, (sum(new) + behind, heads, channels), dtype).float()).to(R.TORCH[dtype])
    starts = torch.tensor([0] + list(new)).cumsum(0).to(torch.int32).cuda()
    return q, starts, caches[0], caches[1], order[:max(shared, 1)].contiguous(), prefix, table, torch.tensor(lengths, dtype=torch.int32, device="cuda")


def check_chunk(odla, lib, case, scale=None, y=None):
    scale = R.scale_of(case[0].shape[-1]) if scale is None else scale
    y = torch.full_like(case[0], 7.0) if y is None else y
    want, tol = P.chunk(*case, scale, y)
    P.call_chunk(odla, lib, *case, scale, y=y)
    P.near(y, want, tol, "chunk")
    return y


CHUNKS = [  # new tokens, own lengths, heads, kv heads, channels, page, prefix
    ([1], [1], 1, 1, 64, 16, 0),
    ([1], [1], 2, 1, 128, 16, 1),
    ([7], [200], 12, 12, 64, 16, 0),
    ([300], [300], 8, 2, 128, 16, 0),
    ([129, 1, 0, 64, 3], [129, 700, 55, 64, 515], 8, 2, 128, 24, 130),
    ([5, 40, 1], [3, 40, 0], 4, 2, 64, 16, 0),            # more new tokens than positions: the first see nothing
    ([5, 1], [2, 0], 4, 2, 64, 16, 20),
    ([256, 255, 257], [256, 511, 900], 4, 4, 64, 32, 0),
    ([70, 33], [1000, 33], 16, 1, 128, 64, 600),
    ([500], [2100], 28, 4, 128, 100, 0),
    ([31, 2, 90], [31, 402, 127], 6, 3, 64, 7, 33),
    ([1] * 40, [(i * 37) % 300 + 1 for i in range(40)], 8, 1, 128, 16, 200),
    ([64], [5000], 32, 8, 128, 16, 0),
    ([3], [9000], 8, 8, 64, 128, 0),
    ([2, 600, 1], [2500, 700, 1], 40, 8, 128, 8, 64),
    ([17, 0, 0, 128], [17, 10, 0, 128], 64, 2, 64, 48, 1),
    ([1024], [1024], 4, 1, 128, 64, 0),
    ([1000, 24], [1500, 2000], 20, 4, 64, 40, 77),
    ([3, 2], [50, 400], 192, 1, 64, 16, 0),               # more heads in a group than a tile has rows, and groups that leave many of its rows empty
    ([9], [300], 100, 1, 128, 24, 10),
    ([140], [300], 36, 2, 128, 256, 0),
]


@pytest.mark.parametrize("dtype", [1, 2])
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("shape", CHUNKS)
def test_chunk(odla, gpu_lib, dtype, token_major, shape):
    check_chunk(odla, gpu_lib, chunk_case(dtype, *shape, token_major=token_major))


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.5])
@pytest.mark.parametrize("dtype,channels", [(1, 128), (2, 64)])
def test_chunk_scales_and_extreme_scores(odla, gpu_lib, dtype, channels, scale):
    """Any scale; positions that outweigh all others by hundreds of units wherever they lie."""
    case = chunk_case(dtype, [140, 9], [400, 9], 4, 1, channels, 16, 150, q_scale=4.0)
    q, starts, kc, vc, pp, prefix, table, lengths = case
    kc[int(table[0, 20]), 0, 3] = q[100, 1] * 3
    kc[int(pp[2]), 0, 7] = q[60, 0] * 3
    check_chunk(odla, gpu_lib, case, scale=scale)


def test_chunk_growing_scores(odla, gpu_lib):
    """Scores that rise step after step, by more and by less than a weight's room, so that the largest changes all the time."""
    for rise in (0.02, 0.3):
        case = chunk_case(2, [200], [900], 2, 1, 64, 16, 0, poison=False)
        q, starts, kc, vc, pp, prefix, table, lengths = case
        q[:] = 1.0
        for i in range(900):
            kc[int(table[0, i // 16]), 0, i % 16] = rise * i / 8
        check_chunk(odla, gpu_lib, case)


@pytest.mark.parametrize("dtype", [1, 2])
@pytest.mark.parametrize("new,heads,kv,channels,page", [([40, 3], 4, 2, 64, 16), ([300, 130], 4, 1, 128, 32), ([300, 130], 4, 4, 64, 7), ([130, 700], 8, 8, 128, 64)])
def test_chunk_a_later_tokens_infinity_stays_its_own(odla, gpu_lib, dtype, new, heads, kv, channels, page):
    """Keys and values of a token that are infinite or no numbers: the tokens before it know nothing of them, itself and those behind do."""
    case = chunk_case(dtype, new, [n + 60 for n in new], heads, kv, channels, page, 0, behind=0)
    q, starts, kc, vc, pp, prefix, table, lengths = case
    clean = R.scale_of(channels)
    want, tol = P.chunk(*case, clean, torch.zeros_like(q))
    where = [(b, n // 2) for b, n in enumerate(new)] + [(b, n - 1) for b, n in enumerate(new)]
    for b, i in where:
        p = 60 + i
        vc[int(table[b, p // page]), :, p % page, :channels // 2] = INF
        vc[int(table[b, p // page]), :, p % page, channels // 2] = float("nan")
    y = P.call_chunk(odla, gpu_lib, *case, clean)
    for b, n in enumerate(new):
        lo = int(starts[b])
        P.near(y[lo:lo + n // 2], want[lo:lo + n // 2], tol[lo:lo + n // 2], "before")
        P.near(y[lo:lo + n, :, channels // 2 + 1:], want[lo:lo + n, :, channels // 2 + 1:], tol[lo:lo + n, :, channels // 2 + 1:], "other channels")
        assert (y[lo + n // 2:lo + n, :, :channels // 2] == INF).all() and y[lo + n // 2:lo + n, :, channels // 2].isnan().all()
    vc.nan_to_num_(nan=0.25, posinf=0.25)
    want, tol = P.chunk(*case, clean, torch.zeros_like(q))
    for b, n in enumerate(new):
        p = 60 + n - 1
        kc[int(table[b, p // page]), :, p % page] = float("nan")      # only the last token sees it
    y = P.call_chunk(odla, gpu_lib, *case, clean)
    for b, n in enumerate(new):
        lo, hi = int(starts[b]), int(starts[b + 1])
        P.near(y[lo:hi - 1], want[lo:hi - 1], tol[lo:hi - 1], "before a key that is no number")
        assert y[hi - 1].isnan().all()


@pytest.mark.parametrize("dtype", [1, 2])
@pytest.mark.parametrize("new,channels", [([1, 3, 200], 128), ([130], 64)])
def test_chunk_scores_of_minus_infinity_weigh_nothing(odla, gpu_lib, dtype, new, channels):
    case = chunk_case(dtype, new, [n + 300 for n in new], 4, 2, channels, 16, 0, poison=False, behind=0)
    q, starts, kc, vc, pp, prefix, table, lengths = case
    q[..., 0] = 1.0
    kc[..., 0] = -INF
    assert (P.call_chunk(odla, gpu_lib, *case, 0.125) == 0).all()
    for b in range(len(new)):
        kc[int(table[b, 9]), :, 5, 0] = 0.0
    y = P.call_chunk(odla, gpu_lib, *case, 0.125)
    for b, n in enumerate(new):
        want = vc[int(table[b, 9]), :, 5].repeat_interleave(2, 0).expand(n, 4, channels)
        assert torch.equal(y[int(starts[b]):int(starts[b + 1])], want)      # (w v) / w, twice rounded in 32 bits


@pytest.mark.parametrize("prefix", [0, 90, 700])
@pytest.mark.parametrize("page", [16, 24])
def test_chunk_bad_pages_are_not_seen(odla, gpu_lib, prefix, page):
    case = chunk_case(2, [30, 1, 130, 2], [100, 300, 250, 90], 8, 1, 128, page, prefix)
    q, starts, kc, vc, pp, _, table, lengths = case
    table[0, 2], table[1, :], table[2, 0], lengths[3] = -1, 1 << 30, kc.shape[0], 100000      # the last: longer than its table
    table[3, -1] = table[0, 1]
    table[3][table[3] < 0] = table[0, 0]
    kc.nan_to_num_(nan=0.5), vc.nan_to_num_(nan=0.5)
    if prefix:
        pp[1] = -7
    check_chunk(odla, gpu_lib, case)


@pytest.mark.parametrize("new,cached", [([200], [600]), ([900] * 12, [1000] * 12)])
def test_chunk_a_wait_that_runs_out_gives_nan_and_the_next_call_is_exact(odla, gpu_lib, monkeypatch, new, cached):
    """The hook leaves one unit of the first block's ring unannounced; the products' wait for it ends after 256 attempts."""
    case = chunk_case(1, new, [n + c for n, c in zip(new, cached)], 8, 2, 128, 16, 0, behind=0)
    monkeypatch.setenv("ODLA_B200_TEST_SKIP_STAGE", "1")
    monkeypatch.setenv("ODLA_B200_TEST_SPIN_LIMIT", "256")
    y = P.call_chunk(odla, gpu_lib, *case, 0.09)
    torch.cuda.synchronize()
    bad = y.isnan().all(-1)
    assert torch.equal(bad, y.isnan().any(-1)) and 0 < int(bad.sum()) <= 256
    monkeypatch.delenv("ODLA_B200_TEST_SKIP_STAGE")
    monkeypatch.delenv("ODLA_B200_TEST_SPIN_LIMIT")
    check_chunk(odla, gpu_lib, case, scale=0.09)


def test_chunk_sees_nothing(odla, gpu_lib):
    case = list(chunk_case(1, [3, 1, 20], [0, 1, 5], 4, 2, 64, 16, 0))
    case[7][0] = -5
    y = check_chunk(odla, gpu_lib, case)
    assert (y[:3] == 0).all() and (y[4:19] == 0).all() and y[23].abs().max() > 0
    case[6] = torch.zeros((3, 0), dtype=torch.int32, device="cuda")
    y = P.call_chunk(odla, gpu_lib, *case, 0.125)
    assert (y[:24] == 0).all() and (y[24:] == 7).all()


def test_chunk_strides_neighbours_and_in_place(odla, gpu_lib):
    """Queries inside a projection's rows, results inside a wider buffer or over the queries: what lies between stays as it was."""
    case = list(chunk_case(1, [33, 64, 2], [50, 64, 700], 6, 2, 64, 16, 50, behind=4))
    q = case[0]
    wide = torch.full((103, 10, 80), 5.0, dtype=q.dtype, device="cuda")
    wide[:, 2:8, 8:72] = q
    out = torch.full((110, 9, 72), 6.0, dtype=q.dtype, device="cuda")
    case[0] = wide[:, 2:8, 8:72]
    check_chunk(odla, gpu_lib, case, y=out[3:106, 1:7, :64])
    assert (out[102:106] == 6.0).all()
    out[3:106, 1:7, :64] = 6.0
    assert (out == 6.0).all()
    want, tol = P.chunk(*case, 0.125, case[0])
    P.call_chunk(odla, gpu_lib, *case, 0.125, y=case[0])
    P.near(case[0], want, tol, "in place")
    wide[:, 2:8, 8:72] = 5.0
    assert (wide == 5.0).all()


def test_chunk_replays_follow_their_batch(odla, gpu_lib):
    """A captured call reads starts, lengths, tables and queries when it runs: other splits of the same rows, fewer sequences, none."""
    case = chunk_case(2, [100, 1, 60, 30], [400, 900, 60, 2000], 8, 2, 128, 16, 100, behind=9, poison=False)
    q, starts, kc, vc, pp, prefix, table, lengths = case
    y = torch.full_like(q, 7.0)
    graph = captured(lambda: P.call_chunk(odla, gpu_lib, *case, 0.088, y=y))
    for new, own in (([100, 1, 60, 30], [400, 900, 60, 2000]), ([0, 1, 0, 190], [30, 901, 30, 1999]), ([1, 1, 1, 1], [400, 900, 60, 2000]), ([0, 0, 0, 0], [0, 0, 0, 0]),
                     ([50, 50, 50, 50], [50, 50, 50, 50])):
        starts.copy_(torch.tensor([0] + new).cumsum(0))
        lengths.copy_(torch.tensor(own))
        q.mul_(0.9)
        y.fill_(7.0)
        want, tol = P.chunk(*case, 0.088, y)
        graph.replay()
        P.near(y, want, tol, str(new))
        again = torch.full_like(q, 7.0)
        P.call_chunk(odla, gpu_lib, *case, 0.088, y=again)
        assert torch.equal(again, y)


def test_chunk_calls_at_the_same_time(odla, gpu_lib):
    cases = [chunk_case(1, [70, 1, 300], [500, 800, 300], 8, 2, 128, 16, 0, seed=s) for s in range(2)]
    alone = [P.call_chunk(odla, gpu_lib, *c, 0.09) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [torch.full_like(c[0], 7.0) for c in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        for st, c, o in zip(streams, cases, outs):
            with torch.cuda.stream(st):
                P.call_chunk(odla, gpu_lib, *c, 0.09, y=o)
    torch.cuda.synchronize()
    assert all(torch.equal(a, o) for a, o in zip(alone, outs))


def test_chunk_far_pages(odla, gpu_lib):
    """Pages whose offsets pass 32 bits, and page numbers whose bytes do."""
    step = (1 << 28) + 1024
    big = [torch.empty(9 * step + 4096, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    kc, vc = (torch.as_strided(b, (10, 2, 16, 64), (step, 1024, 64, 1)) for b in big)
    g = gen(8)
    for c in (kc, vc):
        c.copy_(randn(g, c.shape, 2))
    table = torch.tensor([[9, 0, 8, 3]], dtype=torch.int32, device="cuda")
    q = randn(g, (40, 4, 64), 2)
    starts, lengths = torch.tensor([0, 40], dtype=torch.int32, device="cuda"), torch.tensor([61], dtype=torch.int32, device="cuda")
    check_chunk(odla, gpu_lib, (q, starts, kc, vc, torch.tensor([9], dtype=torch.int32, device="cuda"), 10, table, lengths))


def test_chunk_agrees_with_the_steps_attention(odla, gpu_lib):
    """The same batch through odla_b200_paged_attention, whose sequences all bring the same number of tokens."""
    for queries in (1, 5, 40):
        case = chunk_case(1, [queries] * 6, [200 + 31 * i for i in range(6)], 8, 2, 128, 16, 150, behind=0)
        q, starts, kc, vc, pp, prefix, table, lengths = case
        want, tol = P.chunk(*case, 0.09, torch.zeros_like(q))
        steps = R.call_attention(odla, gpu_lib, q.view(6, queries, 8, 128), kc, vc, pp, prefix, table, lengths, 0.09)
        P.near(steps.view_as(q), want, tol)
        check_chunk(odla, gpu_lib, case, scale=0.09)


# --------------------------------------------------------------------- log probs ----
def check_log_probs(odla, lib, logits, tokens, top, temperature, what=""):
    got = P.call_log_probs(odla, lib, logits, tokens, top, temperature)
    given, given_tol, entropy, entropy_tol, order, lp, lp_tol = P.log_probs(logits, tokens, top, temperature)
    if given is not None:
        P.near(got[0], given, given_tol, what + " given")
    P.near(got[1], entropy, entropy_tol, what + " entropy")
    assert torch.equal(got[2], order), what
    P.near(got[3], lp, lp_tol, what + " alternatives")
    return got


def logits_of(g, rows, vocab, dtype):
    x = 2.5 * torch.randn((rows, vocab), generator=g, device="cuda")
    x[torch.arange(rows, device="cuda"), torch.randint(0, vocab, (rows,), generator=g, device="cuda")] += 9
    return x.to(R.TORCH[dtype])


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("rows,vocab,given,top", [(1, 1, 1, 1), (3, 5, 2, 20), (1, 30522, 1, 5), (4, 1000, 3, 64), (9, 50257, 1, 10), (64, 32000, 1, 20), (2, 262144, 5, 64), (300, 4096, 1, 0), (2, 128000, 0, 20),
                                                  (1, 131071, 2, 33), (170, 8191, 1, 1), (1, 20000, 600, 3), (33, 150001, 1, 8)])
def test_log_probs(odla, gpu_lib, dtype, rows, vocab, given, top):
    g = gen(dtype, rows, vocab)
    logits = logits_of(g, rows, vocab, dtype)
    tokens = torch.randint(-2, vocab + 2, (rows, given), generator=g, device="cuda").to(torch.int32)
    check_log_probs(odla, gpu_lib, logits, tokens, top, None)
    t = torch.tensor([1.0, 0.3, 2.0, 0.0, -1.0, 0.7], device="cuda")[torch.randint(0, 6, (rows,), generator=g, device="cuda")]
    logits[::2, vocab // 3:] = -INF
    if vocab > 4:
        logits[:, 3] = float("nan")
    check_log_probs(odla, gpu_lib, logits, tokens, top, t, "masked")


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_log_probs_rows_anywhere(odla, gpu_lib, dtype, offset):
    """Rows that begin off 16 bytes, with what must not count around them."""
    for vocab, row in ((1000, 1003), (257, 264), (6, 7), (40000, 40001), (3, 0)):
        g = gen(dtype, vocab)
        wide = torch.full((5 * max(row, 1) + vocab + 8,), INF, dtype=R.TORCH[dtype], device="cuda")
        view = torch.as_strided(wide, (5, vocab), (row, 1), offset)
        if row:
            view.copy_(logits_of(g, 5, vocab, dtype))
        else:
            view[0].copy_(logits_of(g, 1, vocab, dtype)[0])
        check_log_probs(odla, gpu_lib, view, torch.randint(0, vocab, (5, 2), generator=g, device="cuda").to(torch.int32), min(vocab, 9), None, "%d" % vocab)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("rows,vocab", [(1, 128000), (5, 30000), (200, 3000), (150, 128000)])
def test_log_probs_equal_logits(odla, gpu_lib, dtype, rows, vocab):
    """Ties by the thousand: all equal, two values, a few, rising and falling; the lower index comes first."""
    i = torch.arange(vocab, device="cuda")
    for what, x in (("equal", torch.full((vocab,), 1.5, device="cuda")), ("two", (i % 7 == 3).float()), ("five", (i * 7919 % 5).float()), ("rising", i.float() / 64), ("falling", -i.float() / 64),
                    ("lowest", torch.full((vocab,), torch.finfo(R.TORCH[dtype]).min, device="cuda")), ("halves", (i // 64 % 2).float()), ("zeros", torch.where(i % 2 == 0, 0.0, -0.0))):
        logits = x.to(R.TORCH[dtype]).expand(rows, vocab).contiguous()
        tokens = torch.tensor([[0, vocab - 1]], dtype=torch.int32, device="cuda").expand(rows, 2).contiguous()
        check_log_probs(odla, gpu_lib, logits, tokens, 20, None, what)
        check_log_probs(odla, gpu_lib, logits, tokens, 64, torch.full((rows,), 0.5, device="cuda"), what)


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_log_probs_infinities_and_masks(odla, gpu_lib, dtype):
    g = gen(dtype)
    vocab = 5000
    x = logits_of(g, 8, vocab, dtype)
    x[0] = -INF                                   # nothing left
    x[1] = float("nan")
    x[2, 17], x[2, 4000], x[2, 4001] = INF, INF, INF
    x[3], x[3, 4999] = -INF, 2.0                  # one left
    x[4, 1:] = torch.finfo(x.dtype).min           # a mask of the type's lowest value
    x[5], x[5, 77] = torch.finfo(x.dtype).min, -INF
    x[6] = torch.finfo(x.dtype).max
    x[7, ::2] = float("nan")
    tokens = torch.tensor([[0, 17, 4999, -1, 5000, 77]], dtype=torch.int32, device="cuda").expand(8, 6).contiguous()
    got = check_log_probs(odla, gpu_lib, x, tokens, 5, None)
    assert got[0][0].isneginf().all() and (got[1][:2] == 0).all() and (got[2][:2] == -1).all()
    assert got[2][2, :3].tolist() == [17, 4000, 4001] and abs(float(got[1][2]) - 1.0986123) < 1e-6 and got[2][3].tolist() == [4999, -1, -1, -1, -1]
    P.call_log_probs(odla, gpu_lib, x, None, 0, None)


def test_log_probs_extreme_temperatures(odla, gpu_lib):
    x = logits_of(gen(4), 6, 3000, 0)
    x[:, 5] = -INF
    t = torch.tensor([1e-30, 1e-3, 1e4, float("nan"), 1e-44, 1e30], device="cuda")
    tokens = torch.randint(0, 3000, (6, 4), generator=gen(5), device="cuda").to(torch.int32)
    check_log_probs(odla, gpu_lib, x[1:4].contiguous(), tokens[1:4].contiguous(), 5, t[1:4].contiguous())
    got = P.call_log_probs(odla, gpu_lib, x, tokens, 5, t)
    assert got[3][0, 0] == 0 and got[3][4, 0] == 0 and (got[1][[0, 4]] == 0).all()
    assert abs(float(got[1][5]) - float(torch.tensor(2999.0).log())) < 1e-4


def test_log_probs_follow_the_sampler_and_replays(odla, gpu_lib):
    """A step: tokens are sampled and their log probabilities taken, in one captured graph that follows its logits."""
    g = gen(6)
    logits, u = logits_of(g, 20, 50000, 2), torch.rand(20, generator=g, device="cuda")
    tokens = torch.zeros((20, 1), dtype=torch.int32, device="cuda")
    out = []

    def call():
        R.call_sample(odla, gpu_lib, logits, None, None, None, None, u, 2, tokens=tokens.view(-1))
        out[:] = P.call_log_probs(odla, gpu_lib, logits, tokens, 10)
    graph = captured(call)
    for _ in range(3):
        logits.copy_(logits_of(g, 20, 50000, 2))
        graph.replay()
        torch.cuda.synchronize()
        want = P.log_probs(logits, tokens, 10, None)
        P.near(out[0], want[0], want[1])
        assert torch.equal(out[2], want[4])
        again = P.call_log_probs(odla, gpu_lib, logits, tokens, 10)
        assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_log_probs_far_rows(odla, gpu_lib):
    step = (1 << 31) + 7
    big = torch.empty(step + 4096, dtype=torch.float16, device="cuda")
    x = torch.as_strided(big, (2, 4000), (step, 1))
    x.copy_(logits_of(gen(9), 2, 4000, 1))
    check_log_probs(odla, gpu_lib, x, torch.tensor([[5], [9]], dtype=torch.int32, device="cuda"), 7, None)


# ------------------------------------------------------------------- all together ----
@pytest.mark.parametrize("dtype", [1, 2])
def test_a_prompt_and_steps_of_a_small_decoder(odla, gpu_lib, dtype):
    """Two layers, two sequences: prompts in two parts of unlike lengths, then single tokens beside the other's prompt; hidden states and the
    tokens' log probabilities as if every sequence had been computed whole in 64 bits."""
    g = gen(dtype, 77)
    T = R.TORCH[dtype]
    W, H, KH, D, V, page, layers = 256, 4, 2, 64, 700, 16, 2
    total = [75, 150]
    embed = torch.randn((V, W), generator=g, device="cuda").to(T)
    norms = [(1 + 0.1 * torch.randn(W, generator=g, device="cuda")).to(T) for _ in range(2 * layers + 1)]
    heads_w = [(1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(T) for _ in range(2)]
    wq = [(torch.randn((W, (H + 2 * KH) * D), generator=g, device="cuda") / 16).to(T) for _ in range(layers)]
    wo = [(torch.randn((H * D, W), generator=g, device="cuda") / 16).to(T) for _ in range(layers)]
    wm = [(torch.randn((W, W), generator=g, device="cuda") / 16).to(T) for _ in range(layers)]
    text = [torch.randint(0, V, (n + 1,), generator=g, device="cuda") for n in total]
    spec = odla.rotary_spec([10000.0 ** (-i / 32) for i in range(32)])
    width = 10
    order = torch.randperm(2 * width + 2, generator=g, device="cuda").to(torch.int32)
    table = order[:2 * width].view(2, width).contiguous()
    kcs, vcs = ([torch.full((2 * width + 2, KH, page, D), float("nan"), dtype=T, device="cuda") for _ in range(layers)] for _ in range(2))
    got_h, got_lp = [[None] * n for n in total], [[None] * n for n in total]
    done = [0, 0]
    # parts: how many tokens each sequence brings
    for part in ([40, 0], [30, 90], [1, 58], [1, 1], [0, 1], [3, 0]):
        rows = [(b, done[b] + i) for b in range(2) for i in range(part[b])]
        n = len(rows)
        starts = torch.tensor([0, part[0], n], dtype=torch.int32, device="cuda")
        lengths = torch.tensor([done[b] + part[b] for b in range(2)], dtype=torch.int32, device="cuda")
        pos = torch.tensor([[p for _, p in rows]], dtype=torch.int32, device="cuda")
        slots = torch.tensor([int(table[b, p // page]) * page + p % page for b, p in rows], dtype=torch.int64, device="cuda")
        hidden = embed[torch.stack([text[b][p] for b, p in rows])].clone()
        delta = torch.zeros_like(hidden)
        for i in range(layers):
            x = torch.empty_like(hidden)
            assert P.call_norm(odla, gpu_lib, delta[:, None], hidden[:, None], norms[2 * i], hidden[:, None], x[:, None]) == 0
            qkv = (x @ wq[i]).view(n, H + 2 * KH, D)
            for part_of, w in ((qkv[:, :H], heads_w[0]), (qkv[:, H:H + KH], heads_w[1])):
                assert P.call_norm(odla, gpu_lib, part_of, weight=w, y=part_of) == 0
            q, y = torch.empty((n, H, D), dtype=T, device="cuda"), torch.empty((n, H, D), dtype=T, device="cuda")
            cache = R.cache_of(odla, kcs[i], dtype)
            st = qkv.stride(0)
            d = odla.AppendDesc(tokens=n, heads=H, q_token=st, q_head=D, k_token=st, k_head=D, v_token=st, v_head=D, y_token=H * D, y_head=D)
            at = [qkv[0, k].data_ptr() for k in (0, H, H + KH)]
            assert gpu_lib.b200_paged_append(C.byref(cache), kcs[i].data_ptr(), vcs[i].data_ptr(), C.byref(d), C.byref(spec), *at, q.data_ptr(), pos.data_ptr(), slots.data_ptr(), R.stream()) == 0
            P.call_chunk(odla, gpu_lib, q, starts, kcs[i], vcs[i], None, 0, table, lengths, 0.125, y=y)
            delta = y.view(n, H * D) @ wo[i]
            assert P.call_norm(odla, gpu_lib, delta[:, None], hidden[:, None], norms[2 * i + 1], hidden[:, None], x[:, None]) == 0
            delta = x @ wm[i]
        x = torch.empty_like(hidden)
        assert P.call_norm(odla, gpu_lib, delta[:, None], hidden[:, None], norms[-1], hidden[:, None], x[:, None]) == 0
        logits = x @ embed.T
        nxt = torch.stack([text[b][p + 1] for b, p in rows]).to(torch.int32)[:, None].contiguous()
        lp = P.call_log_probs(odla, gpu_lib, logits, nxt, 3)[0]
        for j, (b, p) in enumerate(rows):
            got_h[b][p], got_lp[b][p] = x[j], lp[j, 0]
        done = [done[b] + part[b] for b in range(2)]
    assert done == total

    def norm64(v, w):
        return v / (v.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    for b, n in enumerate(total):
        hidden = embed[text[b][:n]].double()
        p = torch.arange(n, device="cuda")
        for i in range(layers):
            qkv = (norm64(hidden, norms[2 * i]) @ wq[i].double()).view(n, H + 2 * KH, D)
            q, k = norm64(qkv[:, :H], heads_w[0]), norm64(qkv[:, H:H + KH], heads_w[1])
            q, k = (R.turned(t, p[None], [10000.0 ** (-j / 32) for j in range(32)], [0] * 32, False)[0] for t in (q, k))
            k, v = (t.repeat_interleave(H // KH, 1) for t in (k, qkv[:, H + KH:]))
            s = torch.einsum("ihd,jhd->hij", q, k) * 0.125
            s = s.masked_fill(p[None, :] > p[:, None], -INF)
            hidden = hidden + torch.einsum("hij,jhd->ihd", s.softmax(-1), v).reshape(n, H * D) @ wo[i].double()
            hidden = hidden + norm64(hidden, norms[2 * i + 1]) @ wm[i].double()
        x = norm64(hidden, norms[-1])
        lp = (x @ embed.double().T).log_softmax(-1).gather(1, text[b][1:, None])[:, 0]
        # Some dozen roundings to the type in a row for each layer, and no growth in between (norms): a hidden state's relative error stays below
        # 40 of their half steps, a log probability's below 40 of the spread of its logits (16 for 256 channels)
        got = torch.stack(got_h[b]).double()
        assert float((got - x).norm() / x.norm()) < 40 * R.HALF_STEP[dtype]
        assert float((torch.stack(got_lp[b]).double() - lp).abs().max()) < 40 * R.HALF_STEP[dtype] * 16
