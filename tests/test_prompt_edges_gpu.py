"""The norm, attention of a chunk and log probabilities at the edges: drawn shapes, first calls inside a capture, host threads, the same call over and over, caches
beyond 32 bits, results over inputs."""
import os
import random
import subprocess
import sys
import threading

import pytest
import torch

import decode_ref as R
import prompt_ref as P
import test_prompt_gpu as T

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("seed", range(24))
def test_chunk_drawn_shapes(odla, gpu_lib, seed):
    rng = random.Random(seed)
    kv = rng.choice([1, 2, 3, 4])
    heads = kv * rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 33])
    batch = rng.choice([1, 1, 2, 5, 17])
    new = [rng.choice([0, 1, 1, rng.randint(2, 40), rng.randint(40, 400)]) for _ in range(batch)]
    lengths = [n + rng.choice([0, 0, rng.randint(1, 200), rng.randint(200, 3000)]) for n in new]
    case = T.chunk_case(rng.choice([1, 2]), new, lengths, heads, kv, rng.choice([64, 128]), rng.choice([8, 16, 24, 32, 40, 48, 64, 96, 100, 128, 200, 256, 3]), rng.choice([0, 0, 1, 77, 128, 500]),
                        token_major=rng.random() < 0.5, seed=seed, behind=rng.randint(0, 9))
    T.check_chunk(odla, gpu_lib, case, scale=rng.choice([None, None, None, -0.1]))


@pytest.mark.parametrize("shape", [([64], [3000], 8, 2, 128, 16, 0), ([300, 1, 77], [900, 50, 77], 28, 4, 128, 24, 100), ([500], [500], 4, 4, 64, 64, 0), ([5], [2000], 8, 8, 128, 32, 0),
                                   ([900, 300], [1500, 400], 16, 2, 128, 100, 0)])
def test_chunk_over_and_over_has_the_same_bits(odla, gpu_lib, shape):
    case = T.chunk_case(2, *shape)
    first = P.call_chunk(odla, gpu_lib, *case, 0.09)
    others = [P.call_chunk(odla, gpu_lib, *case, 0.09) for _ in range(40)]
    assert all(torch.equal(first, y) for y in others)


def test_chunk_behind_what_writes_its_inputs(odla, gpu_lib):
    """Queries come out of the norm and lengths out of a copy right in front of each call, with no wait in between; results are read right behind."""
    case = list(T.chunk_case(2, [130, 3], [700, 40], 8, 2, 128, 16, 0, poison=False, behind=0))
    q, starts, kc, vc, pp, prefix, table, lengths = case
    raw = [q.clone() * (i + 1) for i in range(6)]
    normed = torch.empty_like(q)
    outs = []
    for i in range(6):
        assert P.call_norm(odla, gpu_lib, raw[i], y=normed) == 0
        lengths.copy_(torch.tensor([700 - i, 40 + i], device="cuda"))
        y = P.call_chunk(odla, gpu_lib, normed, *case[1:], 0.09)
        total, h = torch.empty_like(y), torch.empty_like(y)
        assert P.call_norm(odla, gpu_lib, y, y, total=total, y=h) == 0
        outs.append((normed.clone(), lengths.clone(), y, total))
    for n, l, y, total in outs:
        want, tol = P.chunk(n, starts, kc, vc, pp, prefix, table, l, 0.09, torch.zeros_like(n))
        P.near(y, want, tol)
        assert torch.equal(total, y + y)


def test_chunk_dense_cache_beyond_32_bits(odla, gpu_lib):
    """Caches of 2.3 thousand million elements, in both orders, pages at both ends."""
    g = T.gen(12)
    for token_major in (False, True):
        shape = (140000, 16, 8, 128) if token_major else (140000, 8, 16, 128)
        big = [torch.empty(shape, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        kc, vc = (b.transpose(1, 2) if token_major else b for b in big)
        numbers = [139999, 0, 70001, 139998, 131072]
        for n in numbers:
            kc[n], vc[n] = T.randn(g, kc[n].shape, 2), T.randn(g, vc[n].shape, 2)
        table = torch.tensor([numbers], dtype=torch.int32, device="cuda")
        q = T.randn(g, (30, 32, 128), 2)
        starts, lengths = torch.tensor([0, 30], dtype=torch.int32, device="cuda"), torch.tensor([77], dtype=torch.int32, device="cuda")
        pick = torch.tensor(numbers, device="cuda")
        y = P.call_chunk(odla, gpu_lib, q, starts, kc, vc, None, 0, table, lengths, 0.09)
        few = torch.arange(5, dtype=torch.int32, device="cuda")[None]
        want, tol = P.chunk(q, starts, kc[pick], vc[pick], None, 0, few, lengths, 0.09, torch.zeros_like(q))
        P.near(y, want, tol)
        del big, kc, vc


def test_calls_from_host_threads(odla, gpu_lib):
    """Each thread on a stream of its own, all three operators at once."""
    cases = [T.chunk_case(1, [70, 1], [500, 900], 8, 2, 128, 16, 0, seed=s) for s in range(3)]
    logits = [T.logits_of(T.gen(s), 9, 30000, 2) for s in range(3)]
    xs = [T.randn(T.gen(s, 1), (50, 1, 1536), 1) for s in range(3)]

    def all_of(i):
        y = torch.empty_like(xs[i])
        assert P.call_norm(odla, gpu_lib, xs[i], y=y) == 0
        return [P.call_chunk(odla, gpu_lib, *cases[i], 0.09), y] + P.call_log_probs(odla, gpu_lib, logits[i], None, 12)
    alone = [all_of(i) for i in range(3)]
    torch.cuda.synchronize()
    failures = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(15):
                    got = all_of(i)
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(alone[i], got))
        except BaseException as e:      # (a thread's own exception would be lost)
            failures.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures


CAPTURED = r"""
import sys
sys.path[:0] = [%r, %r]
import importlib, torch
import prompt_ref as P, test_prompt_gpu as T
pkg = importlib.import_module("heterogeneity-aware-lowering-and-optimization_b200")
odla, lib = pkg.odla, pkg.load()
case = T.chunk_case(1, [40, 3], [900, 100], 8, 2, 128, 16, 0)
logits = T.logits_of(T.gen(1), 3, 50000, 2)
x = T.randn(T.gen(2), (5, 1, 1000), 0)
y, h, out = torch.full_like(case[0], 7.0), torch.empty_like(x), []
def call():
    P.call_chunk(odla, lib, *case, 0.09, y=y)
    out[:] = P.call_log_probs(odla, lib, logits, None, 9)
    assert P.call_norm(odla, lib, x, y=h) == 0
graph = T.captured(call)
graph.replay()
torch.cuda.synchronize()
want, tol = P.chunk(*case, 0.09, torch.full_like(y, 7.0))
P.near(y, want, tol)
assert torch.equal(out[2], P.log_probs(logits, None, 9, None)[4])
want = P.norm(x, None, None, 1e-6, 0.0)[1]
P.near(h, want, P.norm_tolerance(want, 0))
print("captured")
"""


def test_first_calls_inside_a_capture(gpu_lib):
    """A process whose very first calls are captured: nothing in them waits, allocates or asks what a capture forbids."""
    r = subprocess.run([sys.executable, "-c", CAPTURED % (ROOT, os.path.join(ROOT, "tests"))], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("channels", [64, 1000, 4096, 12288, 16392])
def test_norm_results_over_inputs(odla, gpu_lib, dtype, channels):
    for over in ("x", "residual"):
        g = T.gen(dtype, channels)
        x, r = T.randn(g, (700, 1, channels), dtype), T.randn(g, (700, 1, channels), dtype)
        h, want = P.norm(x, r, None, 1e-6, 0.0)
        total, y = (x, r) if over == "x" else (r, x)
        assert P.call_norm(odla, gpu_lib, x, r, None, total, y) == 0
        assert torch.equal(total, h)
        P.near(y, want, P.norm_tolerance(want, dtype))


@pytest.mark.parametrize("seed", range(12))
def test_norm_drawn_shapes(odla, gpu_lib, seed):
    rng = random.Random(seed)
    channels = rng.choice([rng.randint(1, 300), 8 * rng.randint(1, 600), 32 * rng.randint(1, 300), 128 * rng.randint(1, 60)])
    group = rng.choice([channels] + [g for g in (8, 16, 24, 32, 40, 64, 128, 256, 512, 1024) if channels % g == 0])
    heads = rng.choice([1, 1, 3, 8]) if channels <= 1024 else 1
    for rows in (1, rng.randint(2, 40), 1300):
        for quant in (0, 1, 2):
            T.check_norm(odla, gpu_lib, rng.choice([0, 1, 2]), rows, heads, channels, quant, group if quant else 0, residual=rng.random() < 0.5, weight=rng.choice([None, 0, 1, 2]),
                         pad=rng.choice([0, 0, 8, 16, 1]), with_y=quant == 0 or rng.random() < 0.5, seed=seed)


@pytest.mark.parametrize("seed", range(12))
def test_log_probs_drawn_shapes(odla, gpu_lib, seed):
    rng = random.Random(seed)
    rows, vocab, dtype = rng.choice([1, 2, 7, 40, 149, 600]), rng.choice([rng.randint(1, 100), rng.randint(100, 5000), rng.randint(5000, 60000), rng.randint(60000, 262144)]), rng.choice([0, 1, 2])
    rows = max(1, min(rows, 20000000 // vocab))
    g = T.gen(seed, 99)
    logits = T.logits_of(g, rows, vocab, dtype)
    # few different values: ties everywhere
    if rng.random() < 0.5:
        logits = (logits.float() * 2).round().div(2).to(logits.dtype)
    if rng.random() < 0.5:
        logits[:, torch.randint(0, vocab, (max(1, vocab // 3),), generator=g, device="cuda")] = -T.INF
    tokens = torch.randint(0, vocab, (rows, rng.choice([1, 3])), generator=g, device="cuda").to(torch.int32)
    t = None if rng.random() < 0.5 else torch.rand(rows, generator=g, device="cuda") + 0.3
    T.check_log_probs(odla, gpu_lib, logits, tokens, rng.choice([0, 1, 5, 20, 64]), t)


def test_log_probs_over_and_over_have_the_same_bits(odla, gpu_lib):
    for rows in (1, 64, 600):
        logits = T.logits_of(T.gen(rows), rows, 40000, 1)
        first = P.call_log_probs(odla, gpu_lib, logits, torch.zeros((rows, 1), dtype=torch.int32, device="cuda"), 20)
        for _ in range(20):
            again = P.call_log_probs(odla, gpu_lib, logits, torch.zeros((rows, 1), dtype=torch.int32, device="cuda"), 20)
            assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("new,lengths,heads,kv,channels,page,prefix", [
    ([512, 256], [0, 0], 4, 4, 128, 32, 0),                  # whole tiles of tokens that see nothing
    ([700], [100], 8, 8, 64, 16, 0),                         # the first halves of tiles, and the halves of one
    ([300, 128, 700], [44, 0, 700], 8, 2, 128, 16, 0),
    ([112] * 6, [0, 60, 0, 5, 0, 2000], 8, 8, 128, 64, 0),   # few positions for many blocks, behind a wide table
])
def test_chunk_queries_without_positions_leave_zeros(odla, gpu_lib, new, lengths, heads, kv, channels, page, prefix):
    case = T.chunk_case(2, new, lengths, heads, kv, channels, page, prefix, q_scale=100.0)
    y = T.check_chunk(odla, gpu_lib, case)
    at = 0
    for n, own in zip(new, lengths):
        assert (y[at:at + max(0, n - own)] == 0).all()
        at += n
    for _ in range(10):
        assert torch.equal(T.P.call_chunk(odla, gpu_lib, *case, T.R.scale_of(channels), y=torch.full_like(y, 7.0)), y)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("middle", [0.0, 3e4, -3e4, -6.5e4, 1e36, -4e36, 1e38, -3e38])
def test_log_probs_far_from_what_has_no_probability(odla, gpu_lib, dtype, middle):
    """Logits around a middle near either end of their type, between minus infinities, NaN and the type's lowest, hot and cold."""
    if dtype == 1 and abs(middle) > 65504:
        pytest.skip("not a number of fp16")
    g = T.gen(dtype, int(abs(middle)) % 1000003)
    rows, vocab = 9, 5003
    z = T.randn(g, (rows, vocab), 0).double() * (abs(middle) / 64 + 1) + middle
    z = z.clamp(-torch.finfo(R.TORCH[dtype]).max, torch.finfo(R.TORCH[dtype]).max).to(R.TORCH[dtype])
    kind = torch.randint(0, 8, (rows, vocab), generator=g, device="cuda")
    z[kind == 0], z[kind == 1], z[kind == 2] = -float("inf"), float("nan"), torch.finfo(R.TORCH[dtype]).min
    z[3, 100:] = -float("inf")
    z[4, :4000] = -float("inf")
    z[5, :4000] = torch.finfo(R.TORCH[dtype]).min
    temperature = torch.tensor([1.0, 300.0, 1400.0, 1.0, 1.0, 1.0, 1500.0, 1e5, 1e-3], device="cuda")
    tokens = torch.randint(0, vocab, (rows, 40), generator=g, device="cuda", dtype=torch.int32)
    got = P.call_log_probs(odla, gpu_lib, z, tokens, 20, temperature)
    given, given_tol, entropy, entropy_tol, order, lp, lp_tol = P.log_probs(z, tokens, 20, temperature)
    # (what lies half a step or more below the lowest fp32 number rounds to minus infinity: -3.4e38 at a temperature of 1e-3)
    beyond = -torch.finfo(torch.float32).max * (1 + 2.0 ** -25)
    P.near(got[0], torch.where(given < beyond, -float("inf"), given), given_tol, "given")
    P.near(got[1], entropy, entropy_tol, "entropy")
    assert torch.equal(got[2], order)
    P.near(got[3], torch.where(lp < beyond, -float("inf"), lp), lp_tol, "alternatives")


def test_chunk_many_sequences(odla, gpu_lib):
    """More sequences than a block has threads, some without new tokens, one with many."""
    rng = random.Random(5)
    new = [rng.choice([0, 1, 1, 1, 2, 3]) for _ in range(1000)]
    new[900] = 200
    lengths = [n + rng.randint(0, 60) for n in new]
    T.check_chunk(odla, gpu_lib, T.chunk_case(1, new, lengths, 4, 2, 64, 16, 0, poison=False))
    T.check_chunk(odla, gpu_lib, T.chunk_case(2, new[:700] + [70, 0, 0], lengths[:700] + [70, 3, 0], 2, 1, 128, 24, 20, poison=False))


@pytest.mark.parametrize("page", [16, 24])
def test_chunk_lengths_beyond_the_table(odla, gpu_lib, page):
    case = list(T.chunk_case(2, [40, 3, 200], [300, 20, 200], 8, 2, 128, page, 0, poison=False))
    case[6] = case[6].clamp(min=0)          # (every entry a page that is there)
    case[7] = torch.tensor([100000, 2 ** 31 - 1, 333], dtype=torch.int32, device="cuda")
    T.check_chunk(odla, gpu_lib, case)


@pytest.mark.parametrize("dtype", [0, 2])
@pytest.mark.parametrize("rows,vocab,given", [(1, 60000, 1000), (2, 300, 257), (160, 5001, 512), (3, 262144, 300)])
def test_log_probs_of_many_tokens(odla, gpu_lib, dtype, rows, vocab, given):
    g = T.gen(dtype, rows, vocab, given)
    z = T.logits_of(g, rows, vocab, dtype)
    tokens = torch.randint(-2, vocab + 2, (rows, given), generator=g, device="cuda", dtype=torch.int32)
    T.check_log_probs(odla, gpu_lib, z, tokens, 7, torch.full((rows,), 0.8, device="cuda"))
