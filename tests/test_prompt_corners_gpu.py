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
