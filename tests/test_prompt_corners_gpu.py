"""The norm, attention of a chunk and log probabilities where a number leaves its range, a wait is easily left out, or a part of a block falls behind."""
import pytest
import torch

import decode_ref as R
import prompt_ref as P
import test_prompt_gpu as T

pytestmark = pytest.mark.gpu
HOTTEST = 2.0 ** 100      # what temperatures above it count as


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("rows,vocab", [(8, 5003), (8, 30011), (200, 20011)])
def test_log_probs_infinities_at_high_temperatures(odla, gpu_lib, dtype, rows, vocab):
    """Infinities share all probability, however hot the row."""
    g = T.gen(dtype, rows, vocab)
    z = T.logits_of(g, rows, vocab, dtype)
    temperature = torch.tensor([1.0, 1e6, 4e8, 6e8, 1e9, 1e30, HOTTEST, T.INF], device="cuda").repeat(rows // 8)
    at = torch.stack([torch.randperm(vocab, generator=g, device="cuda")[:3] for _ in range(rows)])
    z.scatter_(1, at, T.INF)
    z[::3, at[0, 0]] = T.INF
    z[1::2, ::5] = -T.INF
    z[:, 7] = float("nan")
    tokens = torch.cat([at, torch.randint(0, vocab, (rows, 5), generator=g, device="cuda")], 1).to(torch.int32)
    got = P.call_log_probs(odla, gpu_lib, z, tokens, 6, temperature)
    given, given_tol, entropy, entropy_tol, order, lp, lp_tol = P.log_probs(z, tokens, 6, temperature.clamp(max=HOTTEST))
    P.near(got[0], given, given_tol, "given")
    P.near(got[1], entropy, entropy_tol, "entropy")
    assert torch.equal(got[2], order)
    P.near(got[3], lp, lp_tol, "alternatives")


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("rows", [4, 200])     # rows that several blocks share, and rows of a block each
def test_log_probs_infinities_beside_the_largest_number(odla, gpu_lib, dtype, rows):
    """A finite logit has no probability beside an infinite one, the type's largest number included: in the same piece, another turn of its thread, another thread, another block."""
    vocab, most = 20011, torch.finfo(R.TORCH[dtype]).max
    for infinite, finite in (([9001], [9000, 9003]), ([9001], [9001 - 8192, 9001 - 4096]), ([9001], [9001 + 4096, 9001 + 8192]), ([9001, 9002], [5]), ([3], [19990]), ([20010], [0]), ([9001], range(vocab))):
        z = T.logits_of(T.gen(dtype, rows), rows, vocab, dtype)
        z[:, list(finite)] = most
        z[1::2, list(finite)[-1]] = most * (1 - 2.0 ** -20) if dtype == 0 else most
        z[:, infinite] = T.INF
        tokens = torch.tensor([infinite[:1] + list(finite)[:2] + [7777]], dtype=torch.int32, device="cuda").expand(rows, -1).contiguous()
        for temperature in (None, torch.full((rows,), 1e-3, device="cuda"), torch.full((rows,), HOTTEST, device="cuda")):
            T.check_log_probs(odla, gpu_lib, z, tokens, 4, temperature, str((infinite, temperature is not None)))


@pytest.mark.parametrize("channels", [64, 128])
@pytest.mark.parametrize("heads,kv,scale", [(8, 2, -0.1), (8, 8, 0.0), (33, 1, 0.1), (48, 1, 0.1), (8, 2, 0.1)])
@pytest.mark.parametrize("new,lengths", [([512, 256], [0, 0]), ([700], [100]), ([300, 128, 700], [44, 0, 700]), ([112] * 6, [0, 60, 0, 5, 0, 2000]), ([3, 2, 1], [0, 0, 0])])
def test_chunk_queries_that_are_no_boxes_leave_zeros(odla, gpu_lib, channels, heads, kv, scale, new, lengths):
    """Tokens that see nothing where queries come by plain loads: a scale that is not positive, groups of heads that leave much of half a tile empty, strides of zero."""
    case = list(T.chunk_case(2, new, lengths, heads, kv, channels, 16, 0, q_scale=100.0))
    if (heads, scale) == (8, 0.1):
        case[0] = case[0][:1].expand(case[0].shape)
    y = T.check_chunk(odla, gpu_lib, case, scale=scale)
    at = 0
    for n, own in zip(new, lengths):
        assert (y[at:at + max(0, n - own)] == 0).all()
        at += n
    for _ in range(10):
        assert torch.equal(P.call_chunk(odla, gpu_lib, *case, scale, y=torch.full(y.shape, 7.0, dtype=y.dtype, device="cuda")), y)


@pytest.mark.parametrize("new,cached,heads,kv,channels,page,prefix", [
    ([600], [3000], 4, 1, 128, 16, 0),           # rings of two places
    ([40], [6000], 2, 1, 128, 64, 300),          # of three, and positions that blocks share
    ([300, 1, 77], [900, 2000, 0], 8, 2, 64, 32, 100),
    ([1000] * 4, [1500] * 4, 8, 8, 64, 16, 0),
])
def test_chunk_a_warp_that_comes_late_misses_nothing(odla, gpu_lib, monkeypatch, new, cached, heads, kv, channels, page, prefix):
    """The warp that takes hidden values out of the boxes is held up for several steps' time in front of each step, also of those that hide nothing."""
    case = T.chunk_case(2, new, [n + c for n, c in zip(new, cached)], heads, kv, channels, page, prefix)
    y = T.check_chunk(odla, gpu_lib, case)
    monkeypatch.setenv("ODLA_B200_TEST_LATE_WARP", "1")
    assert torch.equal(T.check_chunk(odla, gpu_lib, case), y)


@pytest.mark.parametrize("dtype", [0, 2])
@pytest.mark.parametrize("rows,heads,channels", [(5, 1, 4096), (700, 1, 4096), (3, 1, 1001), (9, 5, 128), (3000, 4, 64), (2, 1, 32768), (2, 1, 20001), (700, 1, 5)])
def test_norm_squares_beyond_fp32(odla, gpu_lib, dtype, rows, heads, channels):
    """Rows whose squares pass fp32's range at either end, beside rows of ordinary size, without an epsilon and with one."""
    g = T.gen(dtype, rows, channels)
    size = 2.0 ** torch.tensor([0, 70, 126, -70, -120, 60, 10], dtype=torch.float64, device="cuda")[torch.randint(0, 7, (rows, heads, 1), generator=g, device="cuda")]
    size[0, 0], size[-1, -1] = 2.0 ** 125, 2.0 ** -110
    x = ((1 + torch.rand((rows, heads, channels), generator=g, device="cuda").double()) * size * (torch.randint(0, 2, (rows, heads, channels), generator=g, device="cuda") * 2 - 1)).to(R.TORCH[dtype])
    w = (1 + 0.3 * torch.randn(channels, generator=g, device="cuda"))
    for epsilon in (0.0, 1e-6, 1e30):
        y, total = torch.empty_like(x), torch.empty_like(x)
        q, scales = torch.empty(x.shape, dtype=torch.uint8, device="cuda"), torch.empty((rows, heads, 1), device="cuda")
        assert P.call_norm(odla, gpu_lib, x, torch.zeros_like(x), w, total, y, q, scales, 1, channels, epsilon) == 0
        want = P.norm(x, None, w, epsilon, 0.0)[1]
        P.near(y, want, P.norm_tolerance(want, dtype) + 2.0 ** -126, "y")      # (below the smallest normal number of fp32, as much may be lost)
        values, tol = P.eight_bits(want, 1, scales, False)
        P.near(torch.where(scales >= 2.0 ** -119, q.view(torch.int8).double() * scales.double(), values), values, tol + 2.0 ** -126, "8 bits")   # (127 / max |y| beyond fp32: zeros)
        assert torch.equal(total, x)


@pytest.mark.parametrize("channels", [128, 4096])
def test_norm_of_infinities_beside_large_numbers(odla, gpu_lib, channels):
    x = torch.full((4, 1, channels), 3e38, device="cuda")
    x[1, 0, 3], x[2, 0, 5] = T.INF, float("nan")
    y = torch.empty_like(x)
    assert P.call_norm(odla, gpu_lib, x, y=y) == 0
    P.near(y[[0, 3]], torch.ones_like(y[[0, 3]]).double(), torch.full_like(y[[0, 3]], P.NORM).double())
    assert y[1, 0, 3].isnan() and (y[1, 0, :3] == 0).all() and (y[1, 0, 4:] == 0).all() and y[2].isnan().all()


@pytest.mark.parametrize("dtype", [1, 2])
@pytest.mark.parametrize("new,cached,heads,kv,channels,page", [([40, 3], 300, 4, 2, 64, 16), ([700], 300, 8, 8, 128, 32), ([300, 130], 60, 4, 4, 64, 7), ([5], 6000, 8, 2, 128, 16)])
def test_chunk_no_weight_at_all_gives_zeros_whatever_the_values(odla, gpu_lib, dtype, new, cached, heads, kv, channels, page):
    """Scores of minus infinity throughout, values that are infinite or no numbers among those that all tokens see and among those that the later ones do."""
    case = T.chunk_case(dtype, new, [n + cached for n in new], heads, kv, channels, page, 0, poison=False, behind=0)
    q, starts, kc, vc, pp, prefix, table, lengths = case
    q[..., 0] = 1.0
    kc[..., 0] = -T.INF
    for b, n in enumerate(new):
        for p in (3, cached - 1, cached + n // 2, cached + n - 1):
            vc[int(table[b, p // page]), :, p % page, ::3], vc[int(table[b, p // page]), :, p % page, 1::3] = T.INF, float("nan")
    assert (P.call_chunk(odla, gpu_lib, *case, 0.125) == 0).all()
