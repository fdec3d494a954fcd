"""Plain 64-bit forms of the norm, of attention of a chunk and of log probabilities, and helpers that call the library's."""
import ctypes as C
import math

import torch

from decode_ref import HALF_STEP, TORCH, cache_of, ptr, stream

CODE = {v: k for k, v in TORCH.items()}
MOST = {1: 127.0, 2: 448.0}
U = 2.0 ** -24      # half a step of fp32


# -------------------------------------------------------------------------- norm ----
def call_norm(odla, lib, x, residual=None, weight=None, total=None, y=None, quantised=None, scales=None, quant=0, group=0, epsilon=1e-6, offset=0.0):
    """Tensors [rows, heads, channels] with contiguous channels."""
    def steps(name, t):
        return {} if t is None else {name + "_row": t.stride(0), name + "_head": t.stride(1)}
    d = odla.RmsNormDesc(dtype=CODE[x.dtype], weight_dtype=0 if weight is None else CODE[weight.dtype], rows=x.shape[0], heads=x.shape[1], channels=x.shape[2], quant=quant, group=group,
                         epsilon=epsilon, weight_offset=offset, **steps("x", x), **steps("residual", residual), **steps("sum", total), **steps("y", y), **steps("quant", quantised))
    return lib.b200_rms_norm(C.byref(d), ptr(x), ptr(residual), ptr(weight), ptr(total), ptr(y), ptr(quantised), ptr(scales), stream())


def norm(x, residual, weight, epsilon, offset):
    """h as it is stored, and y in 64 bits."""
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    z = h.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if weight is None else weight.double()
    return h, z / (z.square().mean(-1, keepdim=True) + epsilon).sqrt() * (w + offset)


# Squares are summed 32 at most in a thread, then over ten levels of threads; product, mean, epsilon, root and quotient round once each, h * factor *
# (weight + offset) three times: (32 + 10 + 2) / 2 + 4 + 3 < 40 half steps of fp32.
NORM = 40 * U


def norm_tolerance(y, dtype):
    return y.abs() * (HALF_STEP[dtype] * (1 + NORM) + NORM) + (2.0 ** -25 if dtype == 1 else 0.0)


def eight_bits(y, quant, scales, given):
    """Values in 64 bits for scales that fit y's groups ([rows, heads, groups], or one), and how far what 8 bits stand for may be from them."""
    s = scales.double().reshape(1, 1, 1) if given else scales.double()
    s = s.repeat_interleave(y.shape[-1] // s.shape[-1], -1)
    want = y
    if given:
        want = torch.minimum(torch.maximum(y, s * (-128.0 if quant == 1 else -448.0)), s * MOST[quant])
    # half a step, beside y's own error and a product, a quotient and a scale with a rounding each
    half = s * 0.5 if quant == 1 else torch.maximum(want.abs() * 2.0 ** -4, s * 2.0 ** -10)
    return want, half * (1 + 8 * U) + want.abs() * (NORM + 4 * U)


# ------------------------------------------------------------------------- chunk ----
def call_chunk(odla, lib, q, starts, k_cache, v_cache, prefix_pages, prefix, table, lengths, scale, y=None):
    """q [tokens, heads, channels], caches [pages, heads, page_size, channels] (any strides)."""
    dtype = CODE[q.dtype]
    y = torch.full_like(q, 7.0) if y is None else y
    cache = cache_of(odla, k_cache, dtype)
    d = odla.ChunkAttentionDesc(batch=starts.numel() - 1, tokens=q.shape[0], heads=q.shape[1], prefix_length=prefix, table_width=table.shape[1], scale=scale, q_token=q.stride(0),
                                q_head=q.stride(1), y_token=y.stride(0), y_head=y.stride(1))
    rc = lib.b200_chunk_attention(C.byref(cache), ptr(k_cache), ptr(v_cache), C.byref(d), ptr(q), ptr(starts), ptr(prefix_pages), ptr(table), ptr(lengths), ptr(y), stream())
    assert rc == 0
    return y


def chunk(q, starts, k_cache, v_cache, prefix_pages, prefix, table, lengths, scale, into):
    """y in 64 bits (rows of no sequence as they are in `into`), and a bound on the error."""
    H, D = q.shape[1:]
    pages, KH, ps, _ = k_cache.shape
    y, tol = into.double().clone(), torch.zeros(into.shape, dtype=torch.float64, device=q.device)
    eps = HALF_STEP[CODE[q.dtype]]
    starts, lengths = starts.tolist(), lengths.tolist()

    def rows(numbers, n):
        i = torch.arange(n, device=q.device)
        page = numbers[i // ps].long()
        return page, i % ps, (page >= 0) & (page < pages)
    for b in range(len(lengths)):
        lo, hi = starts[b], starts[b + 1]
        count, n = hi - lo, min(max(lengths[b], 0), table.shape[1] * ps)
        if not count:
            continue
        parts = [rows(p, m) for p, m in ((prefix_pages, prefix), (table[b], n)) if m]
        if not parts:
            y[lo:hi] = 0
            continue
        page, at, there = (torch.cat(x) for x in zip(*parts))
        page = torch.where(there, page, 0)
        sees = prefix + (n - count + torch.arange(count, device=q.device) + 1).clamp(min=0)
        seen = (torch.arange(prefix + n, device=q.device) < sees[:, None]) & there
        for h in range(H):
            k, v = (torch.where(there[:, None], c[page, h // (H // KH), at].double(), 0.0) for c in (k_cache, v_cache))
            # what no token sees may be anything
            any_seen = seen.any(0)[:, None]
            k, v = torch.where(any_seen, k, 0.0), torch.where(any_seen, v, 0.0)
            x = q[lo:hi, h].double()
            s = (x @ k.T * scale).masked_fill(~seen, -math.inf)
            top = s.amax(-1, keepdim=True)
            w = (s - top.clamp(min=-1e300)).exp()
            w = torch.where(seen, w, 0.0)
            total = w.sum(-1, keepdim=True)
            p = torch.where(total > 0, w / total, 0.0)
            y[lo:hi, h] = p @ v
            # weights: one rounding each (fp16: at most 2^-25 of the largest for the smallest), the second product's sums in fp32, scores with
            # fp32 sums of D terms, the exponential to 2^-18; the result is rounded once more
            ds = (D + 4) * U * torch.where(seen, x.abs() @ k.abs().T, 0.0).amax(-1, keepdim=True) * abs(scale) + 2.0 ** -18
            m = seen.sum(-1, keepdim=True)
            tol[lo:hi, h] = (p @ v.abs() + y[lo:hi, h].abs()) * (eps + 2 * ds + (m + 64) * U) + eps * y[lo:hi, h].abs()
            if q.dtype == torch.float16:
                tol[lo:hi, h] += m * 2.0 ** -25 / total.clamp(min=1.0) * v.abs().amax(0) + 2.0 ** -25
    return y, tol * 1.01


# --------------------------------------------------------------------- log probs ----
def call_log_probs(odla, lib, logits, tokens=None, top=0, temperature=None, entropy=True, row=None):
    rows, vocab = logits.shape
    given = 0 if tokens is None else tokens.shape[1]
    d = odla.LogProbsDesc(dtype=CODE[logits.dtype], rows=rows, vocab=vocab, given=given, top=top, row=logits.stride(0) if row is None else row)
    new = dict(device=logits.device)
    out = [torch.full((rows, given), 7.0, **new), torch.full((rows,), 7.0, **new) if entropy else None, torch.full((rows, top), -7, dtype=torch.int32, **new), torch.full((rows, top), 7.0, **new)]
    rc = lib.b200_log_probs(C.byref(d), ptr(logits), ptr(temperature), ptr(tokens) if given else None, ptr(out[0]) if given else None, ptr(out[1]), ptr(out[2]) if top else None,
                            ptr(out[3]) if top else None, stream())
    assert rc == 0
    return out


def log_probs(logits, tokens, top, temperature):
    """Log probabilities of the tokens, entropy, alternatives and theirs in 64 bits, and bounds on the errors of the three."""
    z = logits.double()
    z = torch.where(z.isnan(), -math.inf, z)
    rows, vocab = z.shape
    t = torch.ones(rows, 1, dtype=torch.float64, device=z.device) if temperature is None else torch.where(temperature > 0, temperature, 1.0).double()[:, None]
    m = z.amax(-1, keepdim=True)
    live = m > -math.inf
    d = torch.where(z == m, 0.0, (z - m) / t)
    d = torch.where(live, d, -math.inf)
    w = d.exp()
    total = w.sum(-1, keepdim=True)
    some = torch.where(live, total.clamp(min=1.0).log(), 0.0)
    logp = torch.where(d > -math.inf, d - some, -math.inf)
    wd = torch.where(w > 0, w * d, 0.0).sum(-1, keepdim=True) / total.clamp(min=1.0)
    entropy = torch.where(live, some - wd, 0.0)[:, 0]
    # Sums of a few terms by accumulator and batch, of up to 33 batches, of ten levels of threads and CTAs: less than 64 half steps; a weight is good to
    # 2^-22, and for each power of two that it lies below the largest three roundings of its exponent count (16 powers on average, at most);
    # a given value's own quotient two, the logarithm two
    s = (64 + 4 + 3 * 16 + 4) * U
    bound_e = ((some.abs() + wd.abs() + 1) * (s + 16 * U))[:, 0]

    def bound(lp, dd):
        return torch.where(dd > -math.inf, s + dd.abs() * 4 * U + some * 4 * U, 0.0)
    out = []
    if tokens is not None and tokens.shape[1]:
        there = (tokens >= 0) & (tokens < vocab)
        at = tokens.clamp(0, vocab - 1).long()
        out += [torch.where(there, logp.gather(1, at), -math.inf), torch.where(there, bound(None, d.gather(1, at)), 0.0)]
    else:
        out += [None, None]
    order = z.sort(dim=-1, descending=True, stable=True).indices[:, :top]
    best = z.gather(1, order)
    alternatives = torch.where(best > -math.inf, order, -1)
    lp = torch.where(best > -math.inf, logp.gather(1, order), -math.inf)
    if vocab < top:
        alternatives = torch.nn.functional.pad(alternatives, (0, top - vocab), value=-1)
        lp = torch.nn.functional.pad(lp, (0, top - vocab), value=-math.inf)
    bl = torch.zeros_like(lp)
    bl[:, :order.shape[1]] = bound(None, d.gather(1, order))
    return out + [entropy, bound_e, alternatives.to(torch.int32), lp, bl]


def near(got, want, tol, what=""):
    """Infinities equal, numbers within their bound."""
    got = got.double()
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), what
    err = (got - want)[~inf].abs()
    bad = ~(err <= tol[~inf])
    assert not bad.any(), "%s: %d of %d off, worst %g of its bound" % (what, int(bad.sum()), bad.numel(), float((err / tol[~inf].clamp(min=1e-300)).max()))
