"""The operators of a decoder's serving step, as a list of measurable cases.

    rotary      positions with one to three axes turn pairs of channels (odla_b200_rotary)
    append      keys and values go into a paged cache, keys and queries turned on the way (odla_b200_paged_append)
    attention   a batch reads the paged cache; what all its sequences begin with lies there once (odla_b200_paged_attention)
    sample      the next token from logits, temperature, top-k, top-p, min-p and a given random number (odla_b200_sample)

``run`` computes a case from elementary torch operations, or, with ``own`` set, through the library's entry points on
the current stream.  ``exact`` computes it again in 64 bits, written apart from the plain form.

Sampling, for a row of logits l, with T the temperature and ties in favour of the lower index throughout:
a token whose logit is NaN or minus infinity is never chosen (-1 if none is left); T = 0 takes the largest logit.  Otherwise
w = exp((l - max l) / T), and the tokens kept are: the k largest logits (k <= 0: all); of those, in descending order, each
before which less than top_p of their sum of w has passed (top_p >= 1: all); of those, where w >= min_p.  With W the sum
of w over the tokens kept, the choice is the first kept token, by index, at which the running sum of w exceeds u * W (the
first kept token for u = 0, the last one if rounding leaves none).
"""
import ctypes
import importlib
import math

import numpy as np
import torch

own = False

PKG = "heterogeneity-aware-lowering-and-optimization_b200"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}       # dtype argument of the entry points
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
# query heads, key / value heads, channels of a head
HEADS = [(12, 12, 64), (32, 8, 128), (64, 8, 128), (16, 2, 64), (8, 1, 128), (28, 4, 128), (20, 4, 64), (40, 8, 128)]


def listed():
    return [
        # the patches of one small picture (14 x 14 cells), rows and columns as two axes
        {"name": "rotary_picture_f16", "op": "rotary", "dtype": "f16", "batch": 1, "tokens": 196, "heads": 12, "channels": 64, "axes": 2, "interleaved": True, "heads_first": False},
        # a few long clips: time, height and width; queries and keys lie [batch][heads][positions], as an encoder graph splits them
        {"name": "rotary_clips_bf16", "op": "rotary", "dtype": "bf16", "batch": 2, "tokens": 12288, "heads": 16, "channels": 128, "axes": 3, "interleaved": False, "heads_first": True},
        # one step of a padded decoding batch: one new token per sequence
        {"name": "append_step_b64_bf16", "op": "append", "dtype": "bf16", "tokens": 64, "heads": 32, "kv_heads": 8, "channels": 128, "page": 16, "interleaved": False, "token_major": True, "start": 30000},
        # a single sequence in the library's default type
        {"name": "append_step_b1_f32", "op": "append", "dtype": "f32", "tokens": 1, "heads": 12, "kv_heads": 12, "channels": 64, "page": 16, "interleaved": True, "token_major": False, "start": 511},
        # a long prompt far into a conversation
        {"name": "append_prompt_8191_f16", "op": "append", "dtype": "f16", "tokens": 8191, "heads": 32, "kv_heads": 8, "channels": 128, "page": 64, "interleaved": False, "token_major": False, "start": 900000},
        # an online service at low load: few sequences, a short common prompt
        {"name": "attention_b3_f16", "op": "attention", "dtype": "f16", "batch": 3, "queries": 1, "heads": 12, "kv_heads": 12, "channels": 64, "page": 16, "prefix": 200, "own": 317, "token_major": False},
        # an ordinary decoding batch behind a long system prompt
        {"name": "attention_b32_p8192_bf16", "op": "attention", "dtype": "bf16", "batch": 32, "queries": 1, "heads": 32, "kv_heads": 8, "channels": 128, "page": 16, "prefix": 8192, "own": 700, "token_major": True},
        # several drafted tokens per sequence are checked at once
        {"name": "attention_b16_q5_p1999_f16", "op": "attention", "dtype": "f16", "batch": 16, "queries": 5, "heads": 28, "kv_heads": 4, "channels": 128, "page": 24, "prefix": 1999, "own": 2500, "token_major": False},
        # many questions about one long document
        {"name": "attention_b128_p32768_bf16", "op": "attention", "dtype": "bf16", "batch": 128, "queries": 1, "heads": 32, "kv_heads": 8, "channels": 128, "page": 64, "prefix": 32768, "own": 900, "token_major": False},
        # one sequence over an encoder's vocabulary
        {"name": "sample_b1_v30522_f32", "op": "sample", "dtype": "f32", "rows": 1, "vocab": 30522},
        # a decoding batch over a large vocabulary
        {"name": "sample_b64_v128000_bf16", "op": "sample", "dtype": "bf16", "rows": 64, "vocab": 128000},
        # many candidates at once, full-precision logits
        {"name": "sample_b256_v131072_f32", "op": "sample", "dtype": "f32", "rows": 256, "vocab": 131072},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attention", "attention", "sample"])
    heads, kv_heads, channels = rng.choice(HEADS)
    if op == "rotary":
        batch = _log_int(rng, 1, 16)
        most = max(1, 2 * 12288 * 16 * 128 // (batch * heads * channels))
        return {"op": op, "dtype": rng.choice(["f32", "f16", "bf16"]), "batch": batch, "tokens": _log_int(rng, 1, min(12288, most) // 2 + 1), "heads": heads,
                "channels": channels, "axes": rng.randint(1, 3), "interleaved": rng.random() < 0.5, "heads_first": rng.random() < 0.5}
    if op == "append":
        most = 8191 * 48 * 128 // ((heads + 2 * kv_heads) * channels) // 2
        return {"op": op, "dtype": rng.choice(["f32", "f16", "bf16"]), "tokens": _log_int(rng, 1, min(8191, most)), "heads": heads, "kv_heads": kv_heads, "channels": channels,
                "page": rng.choice([8, 16, 24, 32, 64, 100]), "interleaved": rng.random() < 0.5, "token_major": rng.random() < 0.5, "start": _log_int(rng, 1, 1000000)}
    if op == "sample":
        vocab = _log_int(rng, 1000, 150000)
        return {"op": op, "dtype": rng.choice(["f32", "f16", "bf16"]), "rows": _log_int(rng, 1, min(256, 256 * 131072 // vocab // 2)), "vocab": vocab}
    case = {"op": op, "dtype": rng.choice(["f16", "bf16"]), "batch": _log_int(rng, 1, 128), "queries": rng.choice([1, 1, 1, rng.randint(2, 8)]), "heads": heads, "kv_heads": kv_heads,
            "channels": channels, "page": rng.choice([8, 16, 24, 32, 64, 100]), "prefix": rng.choice([0, 1, 1, 1]) * _log_int(rng, 16, 32768), "own": _log_int(rng, 8, 2500),
            "token_major": rng.random() < 0.5}
    case["own"] = max(case["own"], case["queries"])
    top = work(listed()[8])
    while any(work(case)[k] > top[k] for k in top):
        if case["batch"] > 1:
            case["batch"] = case["batch"] // 2
        else:
            case["prefix"] //= 2
    return case


# ------------------------------------------------------------------------- work ----
def work(case):
    c, e = case, SIZE[case["dtype"]]
    if c["op"] == "rotary":
        n, t = c["batch"] * c["tokens"] * c["heads"] * c["channels"], c["batch"] * c["tokens"]
        return {"bytes": 2 * n * e + 4 * t * c["axes"], "flops": 3 * n}
    if c["op"] == "append":
        t, turned, copied = c["tokens"], (c["heads"] + c["kv_heads"]) * c["channels"], c["kv_heads"] * c["channels"]
        return {"bytes": 2 * t * (turned + copied) * e + 12 * t, "flops": 3 * t * turned}
    if c["op"] == "sample":
        # a subtraction, an exponential, a comparison and a sum for each logit
        return {"bytes": c["rows"] * (c["vocab"] * e + 24), "flops": 4 * c["rows"] * c["vocab"]}
    lengths = _lengths(c)
    seen = sum(c["queries"] * c["prefix"] + sum(max(0, n - c["queries"] + j + 1) for j in range(c["queries"])) for n in lengths)
    kv = 2 * (c["prefix"] + sum(lengths)) * c["kv_heads"] * c["channels"] * e
    return {"bytes": kv + 2 * c["batch"] * c["queries"] * c["heads"] * c["channels"] * e + 4 * (_pages(c["prefix"], c["page"]) + sum(_pages(n, c["page"]) + 1 for n in lengths)),
            "flops": 4 * seen * c["heads"] * c["channels"]}


def _pages(n, page):
    return -(-n // page)


def _lengths(c):
    """Own lengths of a batch's sequences: ragged, the longest and a slot without a sequence among them."""
    b, top, q = c["batch"], c["own"], c["queries"]
    n = [max(q, top - (top * i * 7 % (top * b)) // b) if i else top for i in range(b)]
    if b > 4:
        n[3] = 0
    return n


# ------------------------------------------------------------------------ inputs ----
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _frequencies(pairs, base=10000.0):
    return np.power(base, -np.arange(pairs, dtype=np.float64) / pairs)


def _prepare_rotary(c, g):
    b, t, h, d, dt = c["batch"], c["tokens"], c["heads"], c["channels"], DTYPES[c["dtype"]]
    x = torch.randn((b, h, t, d) if c["heads_first"] else (b, t, h, d), generator=g, device="cuda").to(dt)
    # cells of a grid, axis after axis, from somewhere inside a longer sequence
    n = torch.arange(t, device="cuda")[None, :] + torch.randint(0, 1000, (b, 1), generator=g, device="cuda")
    side = max(1, math.isqrt(t) if c["axes"] == 2 else round((t / 4) ** 0.5) if c["axes"] == 3 else 1)
    pos = {1: [n], 2: [n // side, n % side], 3: [n // (side * side), n // side % side, n % side]}[c["axes"]]
    pairs = d // 2
    if c["axes"] == 1:
        axis, freq = np.zeros(pairs, np.uint8), _frequencies(pairs)
    elif c["axes"] == 2:                      # half the pairs for each axis, each with frequencies of its own
        axis, freq = np.repeat(np.arange(2, dtype=np.uint8), pairs // 2), np.tile(_frequencies(pairs // 2, 100.0), 2)
    else:                                     # one series of frequencies, shared out over the axes
        axis, freq = np.repeat(np.arange(3, dtype=np.uint8), [pairs // 4, pairs * 3 // 8, pairs * 3 // 8]), _frequencies(pairs)
    return {"x": x, "positions": torch.stack(pos).to(torch.int32).contiguous(), "axis": axis, "frequency": freq, "y": torch.empty_like(x)}


def _cache(c, g, pages):
    shape = (pages, c["page"], c["kv_heads"], c["channels"]) if c["token_major"] else (pages, c["kv_heads"], c["page"], c["channels"])
    return [torch.randn(shape, generator=g, device="cuda").to(DTYPES[c["dtype"]]) for _ in range(2)]


def _prepare_append(c, g):
    t, h, kh, d = c["tokens"], c["heads"], c["kv_heads"], c["channels"]
    pages = _pages(t, c["page"]) + 5
    kc, vc = _cache(c, g, pages)
    row = torch.randn((t, (h + 2 * kh) * d), generator=g, device="cuda").to(DTYPES[c["dtype"]])
    if t > 256:       # a prompt: consecutive positions on pages in any order
        table = torch.randperm(pages, generator=g, device="cuda")
        n = torch.arange(t, device="cuda") + 3
        slots, pos = table[n // c["page"]] * c["page"] + n % c["page"], c["start"] + torch.arange(t, device="cuda")
    else:             # a step: one token of each sequence, anywhere; a padded batch ends in slots of -1
        slots = torch.randperm(pages * c["page"], generator=g, device="cuda")[:t]
        pos = torch.randint(0, c["start"] + 1, (t,), generator=g, device="cuda")
        if t > 8:
            slots[-2:] = -1
    return {"qkv": row, "key_cache": kc, "value_cache": vc, "slots": slots.to(torch.int64), "positions": pos.to(torch.int32), "frequency": _frequencies(d // 2),
            "q_out": torch.empty((t, h, d), dtype=row.dtype, device="cuda")}


def _prepare_attention(c, g):
    b, q, h, d = c["batch"], c["queries"], c["heads"], c["channels"]
    lengths = _lengths(c)
    width, shared = _pages(c["own"], c["page"]), _pages(c["prefix"], c["page"])
    used = shared + sum(_pages(n, c["page"]) for n in lengths)
    order = torch.randperm(used + 7, generator=g, device="cuda").to(torch.int32)
    table = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    at = shared
    for i, n in enumerate(lengths):
        table[i, :_pages(n, c["page"])] = order[at:at + _pages(n, c["page"])]
        at += _pages(n, c["page"])
    kc, vc = _cache(c, g, used + 7)
    # queries twice as long as keys: scores spread over several units, as those of a trained model do
    x = (2 * torch.randn((b, q, h, d), generator=g, device="cuda")).to(kc.dtype)
    return {"q": x, "key_cache": kc, "value_cache": vc, "prefix_pages": order[:max(shared, 1)].clone(), "table": table,
            "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), "y": torch.empty_like(x)}


def _prepare_sample(c, g):
    r, v = c["rows"], c["vocab"]
    logits = 2.5 * torch.randn((r, v), generator=g, device="cuda")
    # a handful of likely words; every fifth request is bound by a grammar that allows a part of the vocabulary
    likely = torch.randint(0, v, (r, 12), generator=g, device="cuda")
    logits.scatter_add_(1, likely, 8 * torch.rand((r, 12), generator=g, device="cuda"))
    bound = torch.arange(r, device="cuda")[:, None] % 5 == 4
    logits.masked_fill_(bound & (torch.arange(v, device="cuda")[None, :] // 97 % 3 != 0), -math.inf)

    def choose(values):
        return torch.tensor(values, device="cuda")[torch.randint(0, len(values), (r,), generator=g, device="cuda")]
    return {"logits": logits.to(DTYPES[c["dtype"]]), "temperature": choose([0.0, 0.6, 0.8, 1.0, 1.0, 1.3]), "top_k": choose([0, 0, 20, 50, 200, 1000]).to(torch.int32),
            "top_p": choose([1.0, 1.0, 0.7, 0.9, 0.95]), "min_p": choose([0.0, 0.0, 0.02, 0.1]), "uniform": torch.rand(r, generator=g, device="cuda"),
            "tokens": torch.empty(r, dtype=torch.int32, device="cuda")}


def prepare(case, seed):
    state = {"rotary": _prepare_rotary, "append": _prepare_append, "attention": _prepare_attention, "sample": _prepare_sample}[case["op"]](case, _generator(seed))
    state["case"] = case
    if own:
        _bind(state)
    return state


# --------------------------------------------------------------------- plain forms ----
def _turn(x, angle, interleaved):
    """x [..., channels] turned by angle [..., channels / 2] (64 bits: far positions), in 32 bits."""
    cos, sin = angle.cos().float(), angle.sin().float()
    x = x.float()
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)


def _plain_rotary(s, c):
    freq = torch.from_numpy(s["frequency"]).cuda()
    angle = s["positions"].double()[torch.from_numpy(s["axis"]).long().cuda()].permute(1, 2, 0) * freq    # [batch, tokens, pairs]
    angle = angle[:, None] if c["heads_first"] else angle[:, :, None]
    return _turn(s["x"], angle, c["interleaved"]).to(s["x"].dtype)


def _plain_append(s, c):
    t, h, kh, d = c["tokens"], c["heads"], c["kv_heads"], c["channels"]
    q, k, v = s["qkv"].view(t, h + 2 * kh, d).split([h, kh, kh], dim=1)
    angle = s["positions"].double()[:, None, None] * torch.from_numpy(s["frequency"]).cuda()
    q_out, k = (_turn(x, angle, c["interleaved"]).to(x.dtype) for x in (q, k))
    live = s["slots"] >= 0
    page, at = s["slots"][live] // c["page"], s["slots"][live] % c["page"]
    for cache, x in ((s["key_cache"], k), (s["value_cache"], v)):
        if c["token_major"]:
            cache[page, at] = x[live]
        else:
            cache[page, :, at] = x[live]
    return [q_out, s["key_cache"], s["value_cache"]]


def _rows_of(cache, pages, n, token_major):
    """The first n positions on the given pages: [..., n, kv_heads, channels] in 32 bits."""
    x = cache[pages.clamp(min=0).long()]
    x = (x if token_major else x.transpose(-3, -2)).flatten(-4, -3)
    return x[..., :n, :, :].float()


def _plain_attention(s, c):
    b, q, h, kh, d, prefix = c["batch"], c["queries"], c["heads"], c["kv_heads"], c["channels"], c["prefix"]
    x = s["q"].float().view(b, q, kh, h // kh, d).permute(2, 0, 1, 3, 4)                     # [kv_heads, batch, queries, group, channels]
    k, v = (_rows_of(s[n], s["table"], c["own"], c["token_major"]).permute(2, 0, 1, 3) for n in ("key_cache", "value_cache"))
    rows = x.reshape(kh, b, -1, d)
    score = (rows @ k.transpose(-1, -2)).view(kh, b, q, h // kh, -1) / math.sqrt(d)
    last = s["lengths"][:, None] - q + torch.arange(q, device="cuda")                        # the last own position a query sees
    seen = torch.arange(c["own"], device="cuda") <= last[..., None]
    score = score.masked_fill(~seen[None, :, :, None], -math.inf).view(kh, b, -1, c["own"])
    top = score.amax(-1, keepdim=True)
    if prefix:
        kp, vp = (_rows_of(s[n], s["prefix_pages"], prefix, c["token_major"]).transpose(0, 1) for n in ("key_cache", "value_cache"))
        shared = rows.reshape(kh, -1, d) @ kp.transpose(-1, -2) / math.sqrt(d)
        top = torch.maximum(top, shared.amax(-1).view_as(top))
    top = top.clamp(min=-3e38)
    p = (score - top).exp()
    total, y = p.sum(-1, keepdim=True), p @ v
    if prefix:
        p = (shared - top.view(kh, -1, 1)).exp()
        total, y = total + p.sum(-1).view_as(total), y + (p @ vp).view_as(y)
    y = torch.where(total > 0, y / total, torch.zeros_like(y))                               # a query that sees nothing gives zeros
    return y.view(kh, b, q, h // kh, d).permute(1, 2, 0, 3, 4).reshape(b, q, h, d).to(s["q"].dtype)


def _plain_sample(s, c):
    z = s["logits"].double().nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    z, index = z.sort(dim=-1, descending=True, stable=True)
    t = s["temperature"].double()[:, None]
    top = z[:, :1]
    live = z > -math.inf
    w = torch.where(z == top, 1.0, ((z - top) / torch.where(t > 0, t, 1.0)).exp()) * live
    rank = torch.arange(c["vocab"], device="cuda")
    k = s["top_k"].long()[:, None]
    keep = live & ((rank < k) | (k <= 0)) & ((t > 0) | (rank == 0))
    before = (w * keep).cumsum(-1)
    total, before = before[:, -1:], before - w * keep
    p = s["top_p"].double()[:, None]
    keep &= (before < p * total) | (p >= 1) | (rank == 0)
    keep &= w >= s["min_p"].double()[:, None]
    w = torch.zeros_like(w).scatter_(1, index, w * keep)
    keep = torch.zeros_like(keep).scatter_(1, index, keep)
    run = w.cumsum(-1)
    u = s["uniform"].double()[:, None]
    hit = keep & ((run > u * run[:, -1:]) | (u == 0))
    last = (keep * rank).amax(-1)
    token = torch.where(hit.any(-1), hit.to(torch.uint8).argmax(-1), last)
    return torch.where(live.any(-1), token, -1).to(torch.int32)


# -------------------------------------------------------------- the library's calls ----
def _bind(state):
    """What a program sets up once: the library, descriptors, a workspace."""
    pkg = importlib.import_module(PKG)
    odla, lib, c = pkg.odla, pkg.load(), state["case"]
    d, dt = c.get("channels"), CODES[c["dtype"]]
    state["lib"] = lib
    if c["op"] == "rotary":
        t, h = c["tokens"], c["heads"]
        token, head = (d, t * d) if c["heads_first"] else (h * d, d)
        state["spec"] = odla.rotary_spec(state["frequency"], axis=state["axis"], interleaved=c["interleaved"])
        state["desc"] = odla.RotaryDesc(dtype=dt, batch=c["batch"], tokens=t, heads=h, channels=d, x_batch=t * h * d, x_token=token, x_head=head, y_batch=t * h * d, y_token=token,
                                        y_head=head)
    elif c["op"] == "sample":
        state["desc"] = odla.SampleDesc(dtype=dt, rows=c["rows"], vocab=c["vocab"], row=c["vocab"])
    else:
        kh, page = c["kv_heads"], c["page"]
        head, token = (d, kh * d) if c["token_major"] else (page * d, d)
        state["cache"] = odla.PagedCache(dtype=dt, pages=state["key_cache"].shape[0], page_size=page, heads=kh, channels=d, page=page * kh * d, head=head, token=token)
    if c["op"] == "append":
        row, h = state["qkv"].shape[1], c["heads"]
        state["spec"] = odla.rotary_spec(state["frequency"], interleaved=c["interleaved"])
        state["desc"] = odla.AppendDesc(tokens=c["tokens"], heads=h, q_token=row, q_head=d, k_token=row, k_head=d, v_token=row, v_head=d, y_token=h * d, y_head=d)
    if c["op"] == "attention":
        q, h = c["queries"], c["heads"]
        state["desc"] = odla.PagedAttentionDesc(batch=c["batch"], queries=q, heads=h, prefix_length=c["prefix"], table_width=state["table"].shape[1], scale=1 / math.sqrt(d),
                                                q_batch=q * h * d, q_token=h * d, q_head=d, y_batch=q * h * d, y_token=h * d, y_head=d)
        size = lib.b200_paged_attention_workspace(ctypes.byref(state["cache"]), ctypes.byref(state["desc"]))
        state["workspace"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")


def _own(s, c):
    if "lib" not in s:
        _bind(s)
    lib, ref, stream = s["lib"], ctypes.byref, torch.cuda.current_stream().cuda_stream

    def p(name):
        return s[name].data_ptr()
    if c["op"] == "rotary":
        out = s["y"]
        rc = lib.b200_rotary(ref(s["spec"]), ref(s["desc"]), p("x"), p("y"), p("positions"), stream)
    elif c["op"] == "append":
        out = [s["q_out"], s["key_cache"], s["value_cache"]]
        q, step = p("qkv"), c["channels"] * SIZE[c["dtype"]]
        k = q + c["heads"] * step
        rc = lib.b200_paged_append(ref(s["cache"]), p("key_cache"), p("value_cache"), ref(s["desc"]), ref(s["spec"]), q, k, k + c["kv_heads"] * step, p("q_out"), p("positions"),
                                   p("slots"), stream)
    elif c["op"] == "attention":
        out = s["y"]
        rc = lib.b200_paged_attention(ref(s["cache"]), p("key_cache"), p("value_cache"), ref(s["desc"]), p("q"), p("prefix_pages"), p("table"), p("lengths"), p("y"), p("workspace"),
                                      s["workspace"].numel(), stream)
    else:
        out = s["tokens"]
        rc = lib.b200_sample(ref(s["desc"]), p("logits"), p("temperature"), p("top_k"), p("top_p"), p("min_p"), p("uniform"), p("tokens"), stream)
    if rc:
        raise RuntimeError("%s failed with %d" % (c["op"], rc))
    return out


def run(state):
    c = state["case"]
    if own:
        return _own(state, c)
    return {"rotary": _plain_rotary, "append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}[c["op"]](state, c)


# ------------------------------------------------------------------- the definition ----
def _exact_turn(x, angle, interleaved):
    """Pairs of channels as complex numbers times exp(i angle)."""
    pair = x.unflatten(-1, (-1, 2)) if interleaved else x.unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * torch.polar(torch.ones_like(angle), angle))
    return z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)


def _exact_sample(s, c):
    out = []
    arrays = [s[n].double().cpu().numpy() for n in ("logits", "temperature", "top_k", "top_p", "min_p", "uniform")]
    for l, t, k, p, m, u in zip(*arrays):
        ids = np.flatnonzero(l > -np.inf)                     # (NaN compares false)
        if not ids.size:
            out.append(-1)
            continue
        ids = ids[np.argsort(-l[ids], kind="stable")]
        if t == 0:
            out.append(int(ids[0]))
            continue
        ids = ids[:int(k)] if k > 0 else ids
        top = l[ids[0]]
        with np.errstate(invalid="ignore"):
            w = np.where(l[ids] == top, 1.0, np.exp((l[ids] - top) / t))
        if p < 1:
            passed = np.concatenate([[0.0], np.cumsum(w)])
            n = max(1, int(np.searchsorted(passed[:-1], p * passed[-1], side="left")))
            ids, w = ids[:n], w[:n]
        ids = ids[w >= m]
        w = w[w >= m]
        by_index = np.argsort(ids)
        ids, run = ids[by_index], np.cumsum(w[by_index])
        at = 0 if u == 0 else int(np.searchsorted(run, u * run[-1], side="right"))
        out.append(int(ids[min(at, len(ids) - 1)]))
    return torch.tensor(out, dtype=torch.int32)


def _exact_attention(s, c):
    q, h, kh, d, page = c["queries"], c["heads"], c["kv_heads"], c["channels"], c["page"]
    kc, vc = ((x if c["token_major"] else x.transpose(1, 2)).reshape(-1, kh, d) for x in (s["key_cache"], s["value_cache"]))      # one row per slot

    def slots(pages, n):
        i = torch.arange(n, device="cuda")
        return pages.long()[i // page] * page + i % page
    shared = slots(s["prefix_pages"], c["prefix"])
    out = torch.zeros((c["batch"], q, h, d), dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lengths"].tolist()):
        at = torch.cat([shared, slots(s["table"][b], n)])
        k, v = kc[at].double(), vc[at].double()
        for j in range(q):
            m = c["prefix"] + max(0, n - q + j + 1)
            if m:
                x = s["q"][b, j].double().view(kh, h // kh, d)
                p = torch.softmax(torch.einsum("hgd,nhd->hgn", x, k[:m]) / math.sqrt(d), dim=-1)
                out[b, j] = torch.einsum("hgn,nhd->hgd", p, v[:m]).reshape(h, d)
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "sample":
        return _exact_sample(s, c)
    if c["op"] == "attention":
        return _exact_attention(s, c)
    freq = torch.from_numpy(s["frequency"]).cuda()
    if c["op"] == "rotary":
        pos = s["positions"].double()
        angle = torch.stack([pos[int(a)] * f for a, f in zip(s["axis"], freq)], dim=-1)
        x = s["x"].double()
        return _exact_turn(x, angle.unsqueeze(1 if c["heads_first"] else 2).expand(x.shape[:-1] + (x.shape[-1] // 2,)), c["interleaved"])
    h, kh, d = c["heads"], c["kv_heads"], c["channels"]
    x = s["qkv"].double().view(c["tokens"], h + 2 * kh, d)
    turned = x[:, :h + kh]
    turned = _exact_turn(turned, (s["positions"].double()[:, None] * freq)[:, None].expand(-1, h + kh, -1), c["interleaved"])
    out = [turned[:, :h]]
    for name, rows in (("key_cache", turned[:, h:]), ("value_cache", x[:, h + kh:])):
        cache = s[name].double()
        by_slot = cache if c["token_major"] else cache.transpose(1, 2)
        flat = by_slot.reshape(-1, kh, d)
        for lo in range(0, c["tokens"], 1024):
            at, part = s["slots"][lo:lo + 1024], rows[lo:lo + 1024]
            flat[at[at >= 0]] = part[at >= 0]
        flat = flat.view(by_slot.shape)
        out.append(flat if c["token_major"] else flat.transpose(1, 2).contiguous())
    return out
