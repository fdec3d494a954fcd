"""Calls at the edges of what a decoder's entry points allow, against plain 64-bit forms."""
import ctypes as C

import pytest
import torch

import decode_ref as R

pytestmark = pytest.mark.gpu


def check_sample(odla, lib, logits, p, u, dtype):
    """Every row gets a token (call_sample fills them with -7 first), and the rule's."""
    got = R.call_sample(odla, lib, logits, *p, u, dtype).cpu().numpy()
    want = R.sample(logits.double().cpu().numpy(), *[None if x is None else x.cpu().numpy() for x in p], u.cpu().numpy())
    bad = [(i, int(got[i]), int(want[i])) for i in range(len(want)) if got[i] != want[i]]
    assert not bad, bad[:8]


# --------------------------------------------------------------------- sampling ----
@pytest.mark.parametrize("dtype,top", [(0, 1e5), (0, 1e6), (0, 1e9), (0, 1e10), (0, 1e20), (1, 6e4), (2, 1e6), (2, 1e9), (2, 1e10), (2, 1e20)])
@pytest.mark.parametrize("vocab", [1000, 12000])
def test_sample_a_maximum_beside_which_a_temperature_vanishes(odla, gpu_lib, dtype, top, vocab):
    """One token forced far above the others, two equal ones, and one a step of the type below: next to masked logits and NaN in the same 16
    bytes and to ordinary ones.  70 temperatures are less than half a step of 32 bits of the largest logit, or about as much, or more."""
    g = torch.Generator(device="cuda").manual_seed(vocab + dtype)
    us = [2.0 ** -20, 0.1, 0.24, 0.25, 0.3, 0.49, 0.5, 0.7, 0.76, 0.9, 1 - 2.0 ** -24]
    kinds, rows = 4, 4 * len(us)
    x = 3 * torch.randn((rows, vocab), generator=g, device="cuda")
    inf, step = float("inf"), top * torch.finfo(R.TORCH[dtype]).eps
    at = 8 * 37
    for r in range(rows):
        kind = r % kinds
        x[r, at + 3] = top
        x[r, at] = -inf
        x[r, at + 1] = float("nan")
        if kind == 1:
            x[r, vocab - 9] = top
        if kind == 2:
            x[r, at + 2] = top - step
        if kind == 3:
            x[r, :at + 3] = -inf
            x[r, at + 4:] = float("nan")
    u = torch.tensor(us, device="cuda").repeat_interleave(kinds)
    x = x.to(R.TORCH[dtype])

    def full(v, t=torch.float32):
        return torch.full((rows,), v, device="cuda", dtype=t)
    for T in (2e-4, 0.45, 1.0, step / 140, step / 3):
        for p in ((full(T), None, None, None), (full(T), None, None, full(0.05)), (full(T), None, full(0.9), None), (full(T), full(20, torch.int32), None, None),
                  (full(T), full(20, torch.int32), full(0.7), full(0.01))):
            check_sample(odla, gpu_lib, x, p, u, dtype)
    check_sample(odla, gpu_lib, x, (None, None, None, None), u, dtype)


@pytest.mark.parametrize("dtype", [0, 2])
def test_sample_from_two_host_threads(odla, gpu_lib, dtype):
    """Rows of different lengths ask the same kernel for different amounts of shared memory; no thread's call may be refused for the other's."""
    import threading
    g = torch.Generator(device="cuda").manual_seed(dtype)
    jobs = []
    for vocab in (30522, 1000):
        logits = (3 * torch.randn((256, vocab), generator=g, device="cuda")).to(R.TORCH[dtype])
        u = torch.rand(256, generator=g, device="cuda")
        jobs.append((logits, u, R.call_sample(odla, gpu_lib, logits, None, None, None, None, u, dtype), torch.empty(256, dtype=torch.int32, device="cuda"), torch.cuda.Stream()))
    torch.cuda.synchronize()
    refused = [0, 0]

    def work(i):
        logits, u, _, out, stream = jobs[i]
        d = odla.SampleDesc(dtype=dtype, rows=256, vocab=logits.shape[1], row=logits.shape[1])
        args = (C.byref(d), logits.data_ptr(), None, None, None, None, u.data_ptr(), out.data_ptr(), stream.cuda_stream)
        for n in range(1500):
            refused[i] += gpu_lib.b200_sample(*args) != 0
            if n % 100 == 99:
                stream.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert refused == [0, 0]
    for _, _, alone, out, _ in jobs:
        assert torch.equal(out, alone)


# -------------------------------------------------------------------- attention ----
@pytest.mark.parametrize("heads,kv,channels,queries", [(32, 8, 128, 1), (8, 1, 64, 5), (8, 8, 64, 3), (16, 1, 64, 8)])
def test_attention_one_workspace_for_the_largest_call_and_all_smaller_ones(odla, gpu_lib, heads, kv, channels, queries):
    """Sized once, for the largest batch and table; every smaller call has the same bits as with a workspace of its own, and writes nothing behind it."""
    g = torch.Generator(device="cuda").manual_seed(heads + channels)
    page, batch, prefix, width = 16, 48, 700, 40
    pages = 44 + batch * width
    kc, vc = (torch.randn((pages, kv, page, channels), generator=g, device="cuda").half() for _ in range(2))
    q = torch.randn((batch, queries, heads, channels), generator=g, device="cuda").half()
    table = (44 + torch.arange(batch * width, device="cuda").view(batch, width)).to(torch.int32)
    pp = torch.arange(44, dtype=torch.int32, device="cuda")
    lengths = torch.randint(0, width * page + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    cache = R.cache_of(odla, kc, 1)
    n = heads * channels
    d = odla.PagedAttentionDesc(batch=batch, queries=queries, heads=heads, prefix_length=prefix, table_width=width, scale=0.1, q_batch=queries * n, q_token=n, q_head=channels,
                                y_batch=queries * n, y_token=n, y_head=channels)
    size = gpu_lib.b200_paged_attention_workspace(C.byref(cache), C.byref(d))
    room = torch.full((size + (1 << 26),), 85, dtype=torch.uint8, device="cuda")
    for b in (48, 47, 24, 23, 11, 5, 2, 1):
        for w, shared in ((40, 700), (40, 0), (7, 700), (1, 129), (0, 700)):
            args = (q[:b], kc, vc, pp, shared, table[:b, :w].contiguous(), lengths[:b], 0.1)
            own = R.call_attention(odla, gpu_lib, *args)
            y = R.call_attention(odla, gpu_lib, *args, workspace=room[:size])
            assert torch.equal(y, own), (b, w, shared)
    assert (room[size:] == 85).all()


@pytest.mark.parametrize("batch,queries", [(1, 1), (1, 5), (3, 8), (70, 1)])
def test_attention_thousands_of_small_fp16_weights_are_not_lost(odla, gpu_lib, batch, queries):
    """One position in front of 32000 others that weigh 2^-25.02 of it each, below half of the smallest fp16 number; together 2^-10.  Where all
    values are one, so is the average.  Where only the many have a value, 1024, the average is 1024 n w / (1 + n w).

    Bound: a weight may be off by a half step of fp16 relative to it (2^-11), or, where it is held as a subnormal, by 2^-25 of a scale that lies
    2^7 above the largest weight at least: together less than n (w 2^-11 + 2^-32) of the whole, 2^-16.6, far below half a step of fp16 at one."""
    prefix, own, page, D = 32000, 40, 16, 64
    shared, width = prefix // page, -(-own // page)
    pages = shared + batch * width
    q = torch.zeros((batch, queries, 4, D), dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    kc = torch.zeros((pages, 2, page, D), dtype=torch.float16, device="cuda")
    vc = torch.ones_like(kc)
    scale = 25.02 / 32.0 * 0.6931471805599453       # a score of 32 is 25.02 powers of two
    kc[5, :, 3, 0] = 32.0                           # one position of the prefix
    pp = torch.arange(shared, dtype=torch.int32, device="cuda")
    table = (shared + torch.arange(batch * width, device="cuda").view(batch, width)).to(torch.int32)
    lengths = torch.full((batch,), own, dtype=torch.int32, device="cuda")
    y = R.call_attention(odla, gpu_lib, q, kc, vc, pp, prefix, table, lengths, scale)
    assert (y == 1).all(), y.float().aminmax()
    vc.fill_(1024.0)
    vc[5, :, 3] = 0.0
    y = R.call_attention(odla, gpu_lib, q, kc, vc, pp, prefix, table, lengths, scale)
    for j in range(queries):
        n = prefix - 1 + own - queries + j + 1
        w = 2.0 ** -25.02
        want = 1024 * n * w / (1 + n * w)
        # (the scale itself is 32 bits: the exponent of 25 is good to 25 x 2^-23 of a power of two)
        bound = 1024 * n * (w * (2.0 ** -11 + 2.0 ** -17) + 2.0 ** -32) + want * 2.0 ** -11
        assert (y[:, j].double() - want).abs().max() <= bound, (float(y[:, j].min()), want, bound)


# ---------------------------------------------------------------------- turning ----
def pi_digits(digits):
    """pi by Machin's formula, in whole numbers."""
    from decimal import Decimal, getcontext
    getcontext().prec = digits + 20
    one = 10 ** (digits + 10)

    def arctan_inverse(n):
        total = term = one // n
        k, sign = 3, -1
        while term:
            term //= n * n
            total += sign * (term // k)
            k, sign = k + 2, -sign
        return total
    return Decimal(4 * (4 * arctan_inverse(5) - arctan_inverse(239))) / Decimal(one)


def exact_angles(positions, frequencies):
    """position * frequency modulo a turn, in (-pi, pi], as float64 that is good to 2^-53 of itself."""
    from decimal import Decimal
    two_pi = 2 * pi_digits(420)
    out = []
    for p in positions:
        row = []
        for f in frequencies:
            a = (Decimal(int(p)) * Decimal(f)) % two_pi      # (keeps the sign of the product)
            a = a - two_pi if a > two_pi / 2 else a + two_pi if a < -two_pi / 2 else a
            row.append(float(a))
        out.append(row)
    return torch.tensor(out, dtype=torch.float64, device="cuda")


def turn(odla, lib, x, positions, frequency, interleaved=False):
    """x [tokens, 1, channels] in fp32."""
    tokens, _, ch = x.shape
    d = odla.RotaryDesc(dtype=0, batch=1, tokens=tokens, heads=1, channels=ch, x_batch=tokens * ch, x_token=ch, x_head=ch, y_batch=tokens * ch, y_token=ch, y_head=ch)
    y, spec = torch.empty_like(x), odla.rotary_spec(frequency, interleaved=interleaved)
    assert lib.b200_rotary(C.byref(spec), C.byref(d), x.data_ptr(), y.data_ptr(), positions.data_ptr(), R.stream()) == 0
    return y


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_small_angles_keep_their_bits(odla, gpu_lib, interleaved):
    """(0, b) -> (-b sin t, b cos t): the sine of a small angle shows by itself, relative to its own size.

    The angle is good to |position| 2^-65 turns (the frequency's rounding) and 2^-24 of itself, sincospif to a step (2^-23 relative at most), the product to 2^-24."""
    frequency = [10.0 ** -e * s for e in (9, 8, 7, 6, 5, 4, 3, 2) for s in (1, -1)]
    pos = [1, -1, 3, 77, 1000, -4096]
    n = len(frequency)
    b = 1 + torch.rand((len(pos), 1, n), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    x = torch.stack([torch.zeros_like(b), b], -1).flatten(-2) if interleaved else torch.cat([torch.zeros_like(b), b], -1)
    y = turn(odla, gpu_lib, x, torch.tensor(pos, dtype=torch.int32, device="cuda"), frequency, interleaved)
    got = y[..., 0::2] if interleaved else y[..., :n]
    ang = exact_angles(pos, frequency).unsqueeze(1)
    want = -b.double() * ang.sin()
    p = torch.tensor(pos, dtype=torch.float64, device="cuda").abs().view(-1, 1, 1)
    R.close(got, want, want.abs() * 2.0 ** -22 + b.double() * p * 2.0 ** -65 * 6.2832)


def test_rotary_any_finite_frequency(odla, gpu_lib):
    """Frequencies of many turns per position, up to the largest double, at near and far positions: the angle is good to |position| 2^-65 turns."""
    frequency = [0.7, 6.5, 7.3e3, 1e8 + 0.1, 3.7e15, 2.0 ** 53 + 2, 1.3 * 2.0 ** 64, 1e30, 1.2345e100, 8.5e299, 1.7e308, 2.0 ** 1023, 5e-324, 2.0 ** -60]
    frequency += [-f for f in frequency]
    pos = [1, 2, 3, -7, 4097, 2 ** 31 - 1, -2 ** 31]
    n = len(frequency)
    x = torch.randn((len(pos), 1, 2 * n), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    y = turn(odla, gpu_lib, x, torch.tensor(pos, dtype=torch.int32, device="cuda"), frequency)
    ang = exact_angles(pos, frequency).unsqueeze(1)
    a, b, c, s = x[..., :n].double(), x[..., n:].double(), ang.cos(), ang.sin()
    want, size = torch.cat([a * c - b * s, a * s + b * c], -1), (a.abs() + b.abs()).repeat(1, 1, 2)
    p = torch.tensor(pos, dtype=torch.float64, device="cuda").abs().view(-1, 1, 1)
    R.close(y, want, R.turn_tolerance(want, size, 0) + size * p * 2.0 ** -65 * 6.2832)
    # opposite frequencies turn back
    back = turn(odla, gpu_lib, y, torch.tensor(pos, dtype=torch.int32, device="cuda"), [-f for f in frequency])
    R.close(back, x.double(), 4 * R.turn_tolerance(x.double(), size, 0))


# --------------------------------------------------------------------- in place ----
def test_in_place_with_strides_that_no_step_takes(odla, gpu_lib):
    """A single batch entry or token has no stride to step by: results may go in place whatever the two strides say."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((1, 5, 3, 64), generator=g, device="cuda").half()
    pos = torch.arange(5, dtype=torch.int32, device="cuda").view(1, 1, 5) + 9
    f = [10000.0 ** (-i / 32) for i in range(32)]
    spec = odla.rotary_spec(f)
    want, size = R.turned(x, pos, f, [0] * 32, False)
    d = odla.RotaryDesc(dtype=1, batch=1, tokens=5, heads=3, channels=64, x_batch=0, x_token=192, x_head=64, y_batch=960, y_token=192, y_head=64)
    assert gpu_lib.b200_rotary(C.byref(spec), C.byref(d), x.data_ptr(), x.data_ptr(), pos.data_ptr(), R.stream()) == 0
    R.close(x, want, R.turn_tolerance(want, size, 1))
    # one token and one head of it, queries in place inside the projection's row
    row = torch.randn((1, 3, 64), generator=g, device="cuda").half()
    kc, vc = (torch.zeros((2, 1, 4, 64), dtype=torch.float16, device="cuda") for _ in range(2))
    at = torch.tensor([[3]], dtype=torch.int32, device="cuda")
    want, size = R.turned(row, at, f, [0] * 32, False)
    value = row[0, 2].clone()
    slot = torch.tensor([6], device="cuda")
    cache = R.cache_of(odla, kc, 1)
    d = odla.AppendDesc(tokens=1, heads=1, q_token=192, q_head=64, k_token=192, k_head=64, v_token=192, v_head=64, y_token=64, y_head=0)
    p = row.data_ptr()
    assert gpu_lib.b200_paged_append(C.byref(cache), kc.data_ptr(), vc.data_ptr(), C.byref(d), C.byref(spec), p, p + 128, p + 256, p, at.data_ptr(), slot.data_ptr(), R.stream()) == 0
    tol = R.turn_tolerance(want, size, 1)
    R.close(row[:, 0], want[:, 0], tol[:, 0])
    R.close(kc[1, 0, 2], want[0, 1], tol[0, 1])
    assert torch.equal(vc[1, 0, 2], value)


# ------------------------------------------------------------- sizes beyond the usual ----
def random_attention(odla, lib, dtype, batch, queries, heads, kv, channels, page, prefix, lengths, seed, token_major=False):
    """Own pages in any order, NaN in every slot that no query sees; against the 64-bit form."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    width, shared = max(-(-max(lengths) // page), 1), -(-prefix // page)
    pages = shared + batch * width + 2
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    pp, table = order[:max(shared, 1)].contiguous(), order[shared:shared + batch * width].view(batch, width).contiguous()
    caches = []
    for _ in range(2):
        full = torch.full((pages, page, kv, channels), float("nan"), device="cuda").to(R.TORCH[dtype])
        for row, n in [(pp, prefix)] + list(zip(table, lengths)):
            for j in range(-(-n // page)):
                m = min(page, n - j * page)
                full[int(row[j]), :m] = torch.randn((m, kv, channels), generator=g, device="cuda").to(full.dtype)
        caches.append((full if token_major else full.transpose(1, 2).contiguous().transpose(1, 2)).transpose(1, 2))
    q = (2 * torch.randn((batch, queries, heads, channels), generator=g, device="cuda")).to(R.TORCH[dtype])
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want, tol = R.attention(q.cpu(), caches[0].cpu(), caches[1].cpu(), pp.cpu(), prefix, table.cpu(), lens.cpu(), R.scale_of(channels))
    y = R.call_attention(odla, lib, q, caches[0], caches[1], pp, prefix, table, lens, R.scale_of(channels))
    R.close(y, want, tol, "attention")


@pytest.mark.parametrize("dtype", [1, 2])
@pytest.mark.parametrize("batch,queries,heads,kv,channels,page,prefix,lengths", [
    (1, 260, 2, 1, 64, 16, 0, [260]), (2, 150, 4, 2, 128, 24, 40, [400, 90]), (1, 129, 3, 3, 64, 64, 300, [1]), (3, 33, 4, 1, 64, 7, 0, [33, 500, 0]), (1, 400, 1, 1, 128, 100, 0, [1100]),
    (2, 1, 256, 1, 64, 16, 0, [700, 40]), (3, 1, 100, 1, 128, 16, 150, [0, 129, 333]), (1, 2, 130, 2, 64, 8, 90, [257]), (1, 1, 1024, 16, 64, 16, 0, [200])])
def test_attention_hundreds_of_queries_and_large_groups(odla, gpu_lib, dtype, batch, queries, heads, kv, channels, page, prefix, lengths):
    """More rows of a sequence than two tiles of the tensor cores hold; prompts shorter than their queries; one key head for hundreds of query heads."""
    random_attention(odla, gpu_lib, dtype, batch, queries, heads, kv, channels, page, prefix, lengths, queries + heads, token_major=dtype == 2)


def test_sample_more_rows_than_a_grid_is_high(odla, gpu_lib):
    g = torch.Generator(device="cuda").manual_seed(11)
    logits, u = torch.randn((70001, 5), generator=g, device="cuda"), torch.rand(70001, generator=g, device="cuda")
    check_sample(odla, gpu_lib, logits, (None, torch.full((70001,), 3, dtype=torch.int32, device="cuda"), None, None), u, 0)


@pytest.mark.parametrize("channels,heads", [(1024, 1024), (1023, 600), (2, 1024)])
def test_rotary_the_most_heads_and_channels(odla, gpu_lib, channels, heads):
    g = torch.Generator(device="cuda").manual_seed(channels)
    x = torch.randn((1, 3, heads, channels), generator=g, device="cuda").half()
    y = torch.empty_like(x)
    pos = torch.tensor([[[7, -3, 100]]], dtype=torch.int32, device="cuda")
    pairs = min(128, channels // 2)
    f = [10000.0 ** (-i / pairs) for i in range(pairs)]
    spec, n = odla.rotary_spec(f), heads * channels
    d = odla.RotaryDesc(dtype=1, batch=1, tokens=3, heads=heads, channels=channels, x_batch=3 * n, x_token=n, x_head=channels, y_batch=3 * n, y_token=n, y_head=channels)
    assert gpu_lib.b200_rotary(C.byref(spec), C.byref(d), x.data_ptr(), y.data_ptr(), pos.data_ptr(), R.stream()) == 0
    want, size = R.turned(x, pos, f, [0] * pairs, False)
    R.close(y, want, R.turn_tolerance(want, size, 1))


# -------------------------------------------------------------- one call after another ----
@pytest.mark.parametrize("dtype,rows,vocab", [(0, 300, 1000), (2, 40, 1024), (1, 3, 512)])
def test_a_call_reads_what_the_one_in_front_writes(odla, gpu_lib, dtype, rows, vocab):
    """Turned rows are the logits of the next call, over and over in the same memory with nothing in between: no call may begin to read before the one in front has written."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    n = 24
    x = (3 * torch.randn((n, rows, vocab), generator=g, device="cuda")).to(R.TORCH[dtype])
    pos = torch.randint(0, 1000, (n, rows), generator=g, device="cuda", dtype=torch.int32)
    u = torch.rand((n, rows), generator=g, device="cuda")
    k = torch.full((rows,), 5, dtype=torch.int32, device="cuda")
    spec = odla.rotary_spec([1.0 / (i + 1) for i in range(64)])
    d = odla.RotaryDesc(dtype=dtype, batch=1, tokens=rows, heads=1, channels=vocab, x_batch=rows * vocab, x_token=vocab, x_head=vocab, y_batch=rows * vocab, y_token=vocab, y_head=vocab)

    def turn_into(y, i):
        assert gpu_lib.b200_rotary(C.byref(spec), C.byref(d), x[i].data_ptr(), y.data_ptr(), pos[i].data_ptr(), R.stream()) == 0
    shared, apart = torch.empty_like(x[0]), torch.empty_like(x)
    tokens = torch.full((n, rows), -7, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    for i in range(n):
        turn_into(shared, i)
        R.call_sample(odla, gpu_lib, shared, None, k if i % 2 else None, None, None, u[i], dtype, tokens=tokens[i])
    torch.cuda.synchronize()
    for i in range(n):
        turn_into(apart[i], i)
        torch.cuda.synchronize()
        want = R.sample(apart[i].double().cpu().numpy(), None, k.cpu().numpy() if i % 2 else None, None, None, u[i].cpu().numpy())
        assert (tokens[i].cpu().numpy() == want).all()


@pytest.mark.parametrize("dtype", [1, 2])
@pytest.mark.parametrize("batch,queries,heads,kv,prefix,own", [(40, 1, 8, 2, 500, 90), (6, 5, 8, 1, 300, 400), (2, 70, 4, 1, 0, 300), (3, 1, 4, 4, 40, 70)])
def test_attention_reads_what_the_kernels_in_front_write(odla, gpu_lib, dtype, batch, queries, heads, kv, prefix, own):
    """Caches, tables, lengths and queries change in place between calls with nothing in between: every call has the bits that it has alone."""
    g = torch.Generator(device="cuda").manual_seed(batch)
    page, D, n = 16, 64, 12
    shared, width = -(-prefix // page), -(-own // page)
    pages = shared + batch * width
    sets = []
    for _ in range(n):
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        sets.append([torch.randn((batch, queries, heads, D), generator=g, device="cuda").to(R.TORCH[dtype])] +
                    [torch.randn((pages, kv, page, D), generator=g, device="cuda").to(R.TORCH[dtype]) for _ in range(2)] +
                    [order[:max(shared, 1)].contiguous(), order[shared:].view(batch, width).contiguous(), torch.randint(0, own + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)])
    alone = []
    for q, kc, vc, pp, table, lengths in sets:
        alone.append(R.call_attention(odla, gpu_lib, q, kc, vc, pp, prefix, table, lengths, 0.125))
        torch.cuda.synchronize()
    live = [t.clone() for t in sets[0]]
    size = 1 << 26
    workspace, results = torch.empty(size, dtype=torch.uint8, device="cuda"), [torch.empty_like(sets[0][0]) for _ in range(n)]
    torch.cuda.synchronize()
    for _ in range(3):
        for i in range(n):
            for to, of in zip(live, sets[i]):
                to.copy_(of)
            R.call_attention(odla, gpu_lib, *live[:4], prefix, *live[4:], 0.125, y=results[i], workspace=workspace)
        torch.cuda.synchronize()
        for i in range(n):
            assert torch.equal(results[i], alone[i]), i
            results[i].fill_(7.0)
