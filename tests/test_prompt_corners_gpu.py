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
