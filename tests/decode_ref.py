"""Plain 64-bit forms of the operators of a decoder's serving step, and helpers that call the library's."""
import ctypes as C
import math

import numpy as np
import torch

TORCH = {0: torch.float32, 1: torch.float16, 2: torch.bfloat16}
HALF_STEP = {0: 2.0 ** -24, 1: 2.0 ** -11, 2: 2.0 ** -8}      # of a rounding to the type, relative to the value


def stream():
    return torch.cuda.current_stream().cuda_stream


def turned(x, positions, frequency, axis, interleaved):
    """x [..., tokens, heads, channels] in 64 bits, positions [axes, ..., tokens]: turned, and |a| + |b| of each channel's pair."""
    x = x.double()
    pairs = len(frequency)
    f = torch.tensor(frequency, dtype=torch.float64, device=x.device)
    ang = torch.stack([positions[int(a)].double() for a in axis], -1) * f if pairs else positions[0].double()[..., None][..., :0]
    cos, sin = ang.cos().unsqueeze(-2), ang.sin().unsqueeze(-2)
    a_at = torch.arange(pairs, device=x.device) * (2 if interleaved else 1)
    b_at = a_at + (1 if interleaved else pairs)
    a, b = x[..., a_at], x[..., b_at]
    y, size = x.clone(), torch.zeros_like(x)
    y[..., a_at], y[..., b_at] = a * cos - b * sin, a * sin + b * cos
    size[..., a_at] = size[..., b_at] = a.abs() + b.abs()
    return y, size


def turn_tolerance(y, size, dtype):
    """Cosine and sine come with an error of at most 2^-23 (angle: an eighth of a turn at most, 2^-24 relative; sincospif: two steps),
    the two products and their sum with three roundings of 2^-24; then one rounding to the type."""
    err = size * (2.0 ** -23 + 3 * 2.0 ** -24)
    return err + HALF_STEP[dtype] * (y.abs() + err) + (2.0 ** -25 if dtype == 1 else 0.0)


def attention(q, k_cache, v_cache, prefix_pages, prefix, table, lengths, scale):
    """q [batch, queries, heads, channels], caches [pages, heads, page_size, channels].  Returns y and a bound on the error."""
    B, Q, H, D = q.shape
    pages, KH, ps, _ = k_cache.shape
    y = torch.zeros((B, Q, H, D), dtype=torch.float64)
    tol = torch.zeros_like(y)
    eps = HALF_STEP[{torch.float16: 1, torch.bfloat16: 2}[q.dtype]]

    def rows(table_row, n):
        at = [(int(table_row[i // ps]), i % ps) for i in range(n)]
        at = [(p, i) if 0 <= p < pages else None for p, i in at]
        return at
    for b in range(B):
        n = min(max(int(lengths[b]), 0), len(table[b]) * ps)
        shared, mine = rows(prefix_pages, prefix), rows(table[b], n)
        for j in range(Q):
            at = [x for x in shared + mine[:max(0, n - Q + j + 1)] if x is not None]
            if not at:
                continue
            idx = torch.tensor(at)
            k, v = k_cache[idx[:, 0], :, idx[:, 1]].double(), v_cache[idx[:, 0], :, idx[:, 1]].double()     # [n, KH, D]
            for h in range(H):
                kk, vv, qq = k[:, h // (H // KH)], v[:, h // (H // KH)], q[b, j, h].double()
                s = kk @ qq * scale
                w = (s - s.max()).exp()
                total = w.sum()
                p = w / total
                y[b, j, h] = p @ vv
                # weights: one rounding each (and, in fp16, at most 2^-25 of the largest for the smallest), the second product's sums in fp32,
                # scores with fp32 sums of D terms, the exponential to 2^-21; the result is rounded once more
                av = p @ vv.abs() + y[b, j, h].abs()
                ds = (D + 4) * 2.0 ** -24 * float((kk.abs() @ qq.abs()).max()) * abs(scale) + 2.0 ** -21
                # (a block's weights have its running maximum as reference, so that roundings are relative to each weight)
                tol[b, j, h] = av * (eps + 2 * ds + (len(at) + 64) * 2.0 ** -24) + eps * y[b, j, h].abs() + \
                    (len(at) * 2.0 ** -25 / float(total) * vv.abs().max(0).values + 2.0 ** -25 if q.dtype == torch.float16 else 0.0)
    return y, tol * 1.01


def sample(logits, temperature, top_k, top_p, min_p, uniform):
    """The rule that the header states, row by row in 64 bits.  logits [rows, vocab] as float64; parameters may be None."""
    out = []
    for r in range(logits.shape[0]):
        l = logits[r]
        T = 1.0 if temperature is None else float(temperature[r])
        k = 0 if top_k is None else int(top_k[r])
        P = 1.0 if top_p is None else float(top_p[r])
        m = 0.0 if min_p is None else min(float(min_p[r]), 1.0)
        u = float(uniform[r])
        ids = np.flatnonzero(l > -np.inf)
        if ids.size == 0:
            out.append(-1)
            continue
        ids = ids[np.argsort(-l[ids], kind="stable")]
        if not T > 0:
            out.append(int(ids[0]))
            continue
        if k > 0:
            ids = ids[:k]
        top = l[ids[0]]
        w = np.ones(ids.size)
        other = l[ids] != top
        w[other] = np.exp((l[ids][other] - top) / T)
        if P < 1:
            before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            n = int((before < max(P, 0.0) * w.sum()).sum())
            ids, w = ids[:max(n, 1)], w[:max(n, 1)]
        ids, w = ids[w >= m], w[w >= m]
        order = np.argsort(ids)
        ids, run = ids[order], np.cumsum(w[order])
        if not u > 0:
            out.append(int(ids[0]))
            continue
        hit = np.flatnonzero(run > u * run[-1])
        out.append(int(ids[hit[0] if hit.size else -1]))
    return np.array(out, dtype=np.int32)


def ptr(t):
    return None if t is None else t.data_ptr()


def call_sample(odla, lib, logits, temperature, top_k, top_p, min_p, uniform, dtype, tokens=None, row=None):
    rows, vocab = logits.shape
    d = odla.SampleDesc(dtype=dtype, rows=rows, vocab=vocab, row=logits.stride(0) if row is None else row)
    tokens = torch.full((rows,), -7, dtype=torch.int32, device=logits.device) if tokens is None else tokens
    rc = lib.b200_sample(C.byref(d), ptr(logits), ptr(temperature), ptr(top_k), ptr(top_p), ptr(min_p), ptr(uniform), ptr(tokens), stream())
    assert rc == 0
    return tokens


def cache_of(odla, k_cache, dtype):
    """Caches [pages, heads, page_size, channels] with any strides (channels contiguous)."""
    pages, heads, ps, ch = k_cache.shape
    assert k_cache.stride(3) == 1
    return odla.PagedCache(dtype=dtype, pages=pages, page_size=ps, heads=heads, channels=ch, page=k_cache.stride(0), head=k_cache.stride(1), token=k_cache.stride(2))


def call_attention(odla, lib, q, k_cache, v_cache, prefix_pages, prefix, table, lengths, scale, y=None, workspace=None):
    dtype = {torch.float16: 1, torch.bfloat16: 2}[q.dtype]
    y = torch.full_like(q, 7.0) if y is None else y
    cache = cache_of(odla, k_cache, dtype)
    d = odla.PagedAttentionDesc(batch=q.shape[0], queries=q.shape[1], heads=q.shape[2], prefix_length=prefix, table_width=table.shape[1], scale=scale,
                                q_batch=q.stride(0), q_token=q.stride(1), q_head=q.stride(2), y_batch=y.stride(0), y_token=y.stride(1), y_head=y.stride(2))
    size = lib.b200_paged_attention_workspace(C.byref(cache), C.byref(d))
    assert size >= 0
    if workspace is None:
        workspace = torch.full((max(size, 16),), 255, dtype=torch.uint8, device=q.device)       # NaN everywhere: nothing may rely on it
    rc = lib.b200_paged_attention(C.byref(cache), ptr(k_cache), ptr(v_cache), C.byref(d), ptr(q), ptr(prefix_pages), ptr(table), ptr(lengths), ptr(y), ptr(workspace),
                                  workspace.numel(), stream())
    assert rc == 0
    return y


def close(got, want, tol, what=""):
    err = (got.double().cpu() - want.cpu()).abs()
    bad = ~(err <= tol.cpu())
    assert not bad.any(), "%s %d of %d off, worst %g of its bound" % (what, int(bad.sum()), bad.numel(), float((err / tol.cpu().clamp(min=1e-300)).max()))


def scale_of(channels):
    return 1.0 / math.sqrt(channels)
