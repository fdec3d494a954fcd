"""More operators of a serving decoder, as a list of measurable cases: what a prompt goes through, beside the steps of ``operators.py``.

    norm        root-mean-square norm, with the residual's addition in front and an output in 8 bits behind (odla_b200_rms_norm)
    chunk       attention of a batch's new tokens, of any number for each sequence, over the paged cache (odla_b200_chunk_attention)
    log_probs   log probabilities of given tokens, the entropy and the likeliest alternatives, from logits (odla_b200_log_probs)

``run`` computes a case from elementary torch operations, or, with ``own`` set, through the library's entry points on
the current stream.  ``exact`` computes it again in 64 bits, written apart from the plain form.

Norm, for a row of C channels: h = x + residual, rounded to the storage type; y = h / sqrt(mean(h h) + epsilon) * weight.  In 8 bits a group of
channels (or the whole row) has the scale max |y| / 127 (e4m3: / 448) and the values y / scale, rounded to the nearest; or the scale is given, one for all rows.

Chunk: sequence b has new tokens, rows starts[b] ... starts[b + 1] - 1 of q, and lengths[b] positions of its own, whose last ones the new tokens are, behind a
prefix that all sequences share.  A token sees the prefix and its sequence's positions up to its own.  Rows behind the last sequence's stay as they are.

Log probabilities, for a row of logits l and a temperature T: log p_i = (l_i - max l) / T - log(sum over j of exp((l_j - max l) / T)), minus infinity for a token
that the vocabulary lacks; entropy = -sum of p log p; alternatives in descending order of l, ties in favour of the lower index, -1 where no token is left.
"""
import ctypes
import importlib
import math

import torch

own = False

PKG = "heterogeneity-aware-lowering-and-optimization_b200"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}       # dtype argument of the entry points
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EIGHT = {"none": 0, "s8": 1, "e4m3": 2}       # 8-bit output of the norm
LARGEST = {"s8": 127.0, "e4m3": 448.0}
EPSILON = 1e-6
# query heads, key / value heads, channels of a head
HEADS = [(12, 12, 64), (32, 8, 128), (64, 8, 128), (16, 2, 64), (8, 1, 128), (28, 4, 128), (20, 4, 64), (40, 8, 128)]


def listed():
    return [
        # one token of an encoder's width in the library's default type
        {"name": "norm_b1_f32", "op": "norm", "dtype": "f32", "weight": "f32", "rows": 1, "heads": 1, "channels": 768, "residual": False, "eight": "none", "scales": "none", "group": 768, "plain_out": True},
        # one step of a decoding batch in front of a projection in 8 bits
        {"name": "norm_step_b64_bf16_e4m3", "op": "norm", "dtype": "bf16", "weight": "bf16", "rows": 64, "heads": 1, "channels": 4096, "residual": True, "eight": "e4m3", "scales": "own", "group": 4096,
         "plain_out": False},
        # the query heads of a prompt, inside the projection's rows
        {"name": "norm_heads_4097_bf16", "op": "norm", "dtype": "bf16", "weight": "bf16", "rows": 4097, "heads": 32, "channels": 128, "residual": False, "eight": "none", "scales": "none", "group": 128,
         "plain_out": True},
        # a long prompt in front of a projection in 8 bits, a scale for each 128 channels
        {"name": "norm_prompt_8191_f16_s8", "op": "norm", "dtype": "f16", "weight": "f32", "rows": 8191, "heads": 1, "channels": 5120, "residual": True, "eight": "s8", "scales": "own", "group": 128,
         "plain_out": True},
        # a few words after a short conversation
        {"name": "chunk_b1_n7_f16", "op": "chunk", "dtype": "f16", "batch": 1, "new": 7, "cached": 193, "heads": 12, "kv_heads": 12, "channels": 64, "page": 16, "prefix": 0, "token_major": False},
        # a continuous batch: some sequences decode, others bring parts of their prompts, behind a common system prompt
        {"name": "chunk_b24_n500_f16", "op": "chunk", "dtype": "f16", "batch": 24, "new": 500, "cached": 1500, "heads": 28, "kv_heads": 4, "channels": 128, "page": 24, "prefix": 700, "token_major": True},
        # a question about a document that the cache holds
        {"name": "chunk_b1_n64_c32768_bf16", "op": "chunk", "dtype": "bf16", "batch": 1, "new": 64, "cached": 32768, "heads": 32, "kv_heads": 8, "channels": 128, "page": 16, "prefix": 0,
         "token_major": False},
        # the second half of a long prompt
        {"name": "chunk_b1_n8192_c8192_bf16", "op": "chunk", "dtype": "bf16", "batch": 1, "new": 8192, "cached": 8192, "heads": 32, "kv_heads": 8, "channels": 128, "page": 64, "prefix": 0,
         "token_major": False},
        # one sequence over an encoder's vocabulary
        {"name": "log_probs_b1_v30522_f32", "op": "log_probs", "dtype": "f32", "rows": 1, "vocab": 30522, "given": 1, "top": 5, "scaled": False},
        # the sampled tokens of a decoding batch over a large vocabulary
        {"name": "log_probs_b64_v128000_bf16", "op": "log_probs", "dtype": "bf16", "rows": 64, "vocab": 128000, "given": 1, "top": 20, "scaled": True},
        # a prompt's own tokens
        {"name": "log_probs_prompt_2047_v50257_f16", "op": "log_probs", "dtype": "f16", "rows": 2047, "vocab": 50257, "given": 1, "top": 1, "scaled": False},
        # several candidates for each position of a long text, full-precision logits
        {"name": "log_probs_1024_v131072_f32", "op": "log_probs", "dtype": "f32", "rows": 1024, "vocab": 131072, "given": 8, "top": 10, "scaled": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _scores(c):
    """Scores of the padded batch, which the plain form holds."""
    return c["batch"] * c["heads"] * c["new"] * (c["new"] + c["cached"] + c["prefix"])


def draw(rng):
    op = rng.choice(["norm", "chunk", "log_probs"])
    top = {c["op"]: c for c in listed()}                      # the last listed of each is its largest
    top["norm"] = listed()[3]
    top["chunk"] = listed()[7]
    most = work(top[op])
    if op == "norm":
        heads = rng.choice([1, 1, rng.choice([8, 12, 28, 32, 40])])
        channels = rng.choice([64, 128]) if heads > 1 else rng.choice([_log_int(rng, 100, 8192), 8 * _log_int(rng, 16, 1024), 768, 1024, 2048, 3584, 4096, 5120, 8192])
        eight = rng.choice(["none", "s8", "e4m3"])
        group = rng.choice([channels] + [g for g in (32, 64, 128) if channels % g == 0])
        case = {"op": op, "dtype": rng.choice(["f32", "f16", "bf16"]), "weight": "f32", "rows": _log_int(rng, 1, 8191), "heads": heads, "channels": channels, "residual": heads == 1 and rng.random() < 0.6,
                "eight": eight, "scales": "none" if eight == "none" else rng.choice(["own", "own", "given"]), "group": group, "plain_out": eight == "none" or rng.random() < 0.5}
        case["weight"] = rng.choice(["f32", case["dtype"]])
        if case["scales"] != "own":
            case["group"] = channels
        size = "rows"
    elif op == "log_probs":
        case = {"op": op, "dtype": rng.choice(["f32", "f16", "bf16"]), "rows": _log_int(rng, 1, 2048), "vocab": _log_int(rng, 1000, 150000), "given": rng.choice([0, 1, 1, rng.randint(2, 16)]),
                "top": rng.choice([0, 1, rng.randint(2, 20), rng.randint(2, 20)]), "scaled": rng.random() < 0.5}
        size = "rows"
    else:
        heads, kv_heads, channels = rng.choice(HEADS)
        case = {"op": op, "dtype": rng.choice(["f16", "bf16"]), "batch": _log_int(rng, 1, 32), "new": _log_int(rng, 1, 8192), "cached": rng.choice([0, 1, 1]) * _log_int(rng, 16, 32768), "heads": heads,
                "kv_heads": kv_heads, "channels": channels, "page": rng.choice([8, 16, 24, 32, 64, 100]), "prefix": rng.choice([0, 0, 1]) * _log_int(rng, 16, 4096), "token_major": rng.random() < 0.5}
        while _scores(case) > _scores(top[op]):
            size = "batch" if case["batch"] > 1 else "new" if case["new"] > 64 else "cached"
            case[size] //= 2
        size = "new"
    while any(work(case)[k] > most[k] for k in most) and case[size] > 1:
        case[size] //= 2
    return case


# ------------------------------------------------------------------------- work ----
def work(case):
    c, e = case, SIZE[case["dtype"]]
    if c["op"] == "norm":
        n = c["rows"] * c["heads"] * c["channels"]
        scales = 4 * n // c["group"] if c["scales"] == "own" else 4
        return {"bytes": n * (e * (1 + 2 * c["residual"] + c["plain_out"]) + (c["eight"] != "none")) + c["channels"] * SIZE[c["weight"]] + (scales if c["eight"] != "none" else 0),
                "flops": n * (4 + c["residual"] + 2 * (c["eight"] != "none"))}
    if c["op"] == "log_probs":
        # a subtraction, a scaling, an exponential and two sums for each logit
        return {"bytes": c["rows"] * (c["vocab"] * e + 8 * c["given"] + 8 * c["top"] + 4 + 4 * c["scaled"]), "flops": 5 * c["rows"] * c["vocab"]}
    new, lengths = _lengths(c)
    seen = sum(n * (c["prefix"] + m - n) + n * (n + 1) // 2 for n, m in zip(new, lengths))
    used = [m if n else 0 for n, m in zip(new, lengths)]
    kv = 2 * (c["prefix"] + sum(used)) * c["kv_heads"] * c["channels"] * e
    return {"bytes": kv + 2 * sum(new) * c["heads"] * c["channels"] * e + 4 * (_pages(c["prefix"], c["page"]) + sum(_pages(m, c["page"]) + 2 for m in used)),
            "flops": 4 * seen * c["heads"] * c["channels"]}


def _pages(n, page):
    return -(-n // page)


def _lengths(c):
    """New tokens and own positions of a batch's sequences: the largest first, every third one decodes, one brings nothing."""
    b, n, cached = c["batch"], c["new"], c["cached"]
    new = [n if i == 0 else 1 if i % 3 == 1 else max(1, n - n * (i * 7 % b) // b) for i in range(b)]
    before = [cached if i == 0 else cached - cached * (i * 5 % b) // b for i in range(b)]
    if b > 4:
        new[3] = 0
    return new, [x + y for x, y in zip(new, before)]


# ------------------------------------------------------------------------ inputs ----
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _prepare_norm(c, g):
    rows, heads, ch, dt = c["rows"], c["heads"], c["channels"], DTYPES[c["dtype"]]
    # heads lie inside a projection's rows, which have as many other columns
    x = torch.randn((rows, heads * (2 if heads > 1 else 1), ch), generator=g, device="cuda")
    s = {"weight": (1 + 0.2 * torch.randn(ch, generator=g, device="cuda")).to(DTYPES[c["weight"]])}
    # a few channels of a trained model's hidden state are far larger than the others
    x[..., torch.randint(0, ch, (max(1, ch // 500),), generator=g, device="cuda")] *= 20
    s["x"] = x.to(dt)
    shape = (rows, heads, ch)
    if c["residual"]:
        s["residual"] = (3 * torch.randn(shape, generator=g, device="cuda")).to(dt)
        s["sum"] = torch.empty(shape, dtype=dt, device="cuda")
    if c["plain_out"]:
        s["y"] = torch.empty(shape, dtype=dt, device="cuda")
    if c["eight"] != "none":
        s["eight"] = torch.empty(shape, dtype=torch.int8 if c["eight"] == "s8" else torch.float8_e4m3fn, device="cuda")
        s["scales"] = torch.empty((rows, heads, ch // c["group"]), device="cuda")
        if c["scales"] == "given":                       # as a calibration finds it: most values inside, the largest saturate
            s["scales"] = torch.full((1,), 3.5 / LARGEST[c["eight"]], device="cuda")
    return s


def _prepare_chunk(c, g):
    h, kh, d, page, dt = c["heads"], c["kv_heads"], c["channels"], c["page"], DTYPES[c["dtype"]]
    new, lengths = _lengths(c)
    width, shared = _pages(max(lengths), page), _pages(c["prefix"], page)
    used = shared + sum(_pages(n, page) for n in lengths)
    order = torch.randperm(used + 7, generator=g, device="cuda").to(torch.int32)
    table = torch.full((c["batch"], width), -1, dtype=torch.int32, device="cuda")
    at = shared
    for i, n in enumerate(lengths):
        table[i, :_pages(n, page)] = order[at:at + _pages(n, page)]
        at += _pages(n, page)
    shape = (used + 7, page, kh, d) if c["token_major"] else (used + 7, kh, page, d)
    kc, vc = (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt) for _ in range(2))
    tokens = (sum(new) + 7) // 8 * 8 if c["batch"] > 1 else sum(new)                         # a padded batch
    # queries twice as long as keys: scores spread over several units, as those of a trained model do
    q = (2 * torch.randn((tokens, h, d), generator=g, device="cuda")).to(dt)
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
    return {"q": q, "key_cache": kc, "value_cache": vc, "prefix_pages": order[:max(shared, 1)].clone(), "table": table, "starts": starts,
            "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), "y": torch.zeros_like(q)}


def _prepare_log_probs(c, g):
    r, v = c["rows"], c["vocab"]
    logits = 2.5 * torch.randn((r, v), generator=g, device="cuda")
    # a handful of likely words; every fifth request is bound by a grammar that allows a part of the vocabulary
    likely = torch.randint(0, v, (r, 12), generator=g, device="cuda")
    logits.scatter_add_(1, likely, 8 * torch.rand((r, 12), generator=g, device="cuda"))
    bound = torch.arange(r, device="cuda")[:, None] % 5 == 4
    logits.masked_fill_(bound & (torch.arange(v, device="cuda")[None, :] // 97 % 3 != 0), -math.inf)
    # mostly likely tokens, others anywhere; a padded batch ends in tokens of -1
    tokens = torch.randint(0, v, (r, c["given"]), generator=g, device="cuda")
    tokens[:, :1] = likely[:, :1]
    if r > 8 and c["given"]:
        tokens[-2:] = -1
    s = {"logits": logits.to(DTYPES[c["dtype"]]), "tokens": tokens.to(torch.int32), "given": torch.empty((r, c["given"]), device="cuda"), "entropy": torch.empty(r, device="cuda"),
         "top_tokens": torch.empty((r, c["top"]), dtype=torch.int32, device="cuda"), "top": torch.empty((r, c["top"]), device="cuda")}
    if c["scaled"]:
        s["temperature"] = torch.tensor([0.6, 0.8, 1.0, 1.3], device="cuda")[torch.randint(0, 4, (r,), generator=g, device="cuda")]
    return s


def prepare(case, seed):
    state = {"norm": _prepare_norm, "chunk": _prepare_chunk, "log_probs": _prepare_log_probs}[case["op"]](case, _generator(seed))
    state["case"] = case
    if own:
        _bind(state)
    return state


# --------------------------------------------------------------------- plain forms ----
def _plain_norm(s, c):
    x = s["x"][:, :c["heads"]].float()
    out = []
    if c["residual"]:
        x = (x + s["residual"].float()).to(s["x"].dtype)
        out.append(x)
        x = x.float()
    y = x * (x.square().mean(-1, keepdim=True) + EPSILON).rsqrt() * s["weight"].float()
    if c["plain_out"]:
        out.append(y.to(s["x"].dtype))
    if c["eight"] != "none":
        top = LARGEST[c["eight"]]
        if c["scales"] == "own":
            groups = y.unflatten(-1, (-1, c["group"]))
            scale = groups.abs().amax(-1) / top
            out.append(scale)
            scale = scale[..., None]
        else:
            groups, scale = y[..., None, :], s["scales"]
        q = torch.where(scale > 0, groups / scale, 0.0).clamp(-top - (c["eight"] == "s8"), top)
        if c["eight"] == "s8":
            out.append((q.round() * scale).to(torch.float16).flatten(-2))        # what 8 bits stand for
        else:
            out.append(q.to(torch.float8_e4m3fn).flatten(-2))
    return out


def _rows_of(cache, pages, n, token_major):
    """The first n positions on the given pages: [..., n, kv_heads, channels] in 32 bits."""
    x = cache[pages.clamp(min=0).long()]
    x = (x if token_major else x.transpose(-3, -2)).flatten(-4, -3)
    return x[..., :n, :, :].float()


def _plain_chunk(s, c):
    b, h, kh, d, prefix, new = c["batch"], c["heads"], c["kv_heads"], c["channels"], c["prefix"], c["new"]
    count, longest = s["starts"].diff(), c["new"] + c["cached"]
    i = torch.arange(new, device="cuda")
    at, live = s["starts"][:-1, None] + i, i < count[:, None]                                 # [batch, new]
    x = s["q"][at.clamp(max=s["q"].shape[0] - 1)].float().view(b, new, kh, h // kh, d).permute(2, 0, 1, 3, 4).reshape(kh, b, -1, d)
    k, v = (_rows_of(s[n], s["table"], longest, c["token_major"]).permute(2, 0, 1, 3) for n in ("key_cache", "value_cache"))
    score = (x @ k.transpose(-1, -2)).view(kh, b, new, h // kh, -1).div_(math.sqrt(d))
    last = (s["lengths"] - count)[:, None] + i                                                # the last own position a token sees
    score.masked_fill_(~(torch.arange(k.shape[2], device="cuda") <= last[..., None])[None, :, :, None], -math.inf)
    score = score.view(kh, b, -1, k.shape[2])
    top = score.amax(-1, keepdim=True)
    if prefix:
        kp, vp = (_rows_of(s[n], s["prefix_pages"], prefix, c["token_major"]).transpose(0, 1) for n in ("key_cache", "value_cache"))
        shared = x.view(kh, -1, d) @ kp.transpose(-1, -2) / math.sqrt(d)
        top = torch.maximum(top, shared.amax(-1).view_as(top))
    top = top.clamp(min=-3e38)
    p = score.sub_(top).exp_()
    total, y = p.sum(-1, keepdim=True), p @ v
    if prefix:
        p = (shared - top.view(kh, -1, 1)).exp()
        total, y = total + p.sum(-1).view_as(total), y + (p @ vp).view_as(y)
    y = torch.where(total > 0, y / total, torch.zeros_like(y)).view(kh, b, new, h // kh, d).permute(1, 2, 0, 3, 4).reshape(b, new, h, d).to(s["q"].dtype)
    out = s["y"].clone()
    out[at[live]] = y[live]
    return out


def _plain_log_probs(s, c):
    z = s["logits"].float().nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    top = z.amax(-1, keepdim=True)
    t = s["temperature"][:, None] if c["scaled"] else 1.0
    d = torch.where(z == top, 0.0, (z - top) / t)
    w = d.exp()
    total = w.double().sum(-1, keepdim=True).float()
    some = total.log()
    entropy = some[:, 0] - (torch.where(w > 0, w * d, 0.0).sum(-1) / total[:, 0])
    there = (s["tokens"] >= 0) & (s["tokens"] < c["vocab"])
    given = torch.where(there, d.gather(1, s["tokens"].clamp(0, c["vocab"] - 1).long()) - some, -math.inf)
    best, index = z.sort(dim=-1, descending=True, stable=True)
    best, index = best[:, :c["top"]], index[:, :c["top"]]
    alternatives = d.gather(1, index) - some
    return [given, entropy, torch.where(best > -math.inf, index, -1).to(torch.int32), alternatives]


# -------------------------------------------------------------- the library's calls ----
def _bind(state):
    """What a program sets up once: the library and descriptors."""
    pkg = importlib.import_module(PKG)
    odla, c = pkg.odla, state["case"]
    state["lib"] = pkg.load()
    dt = CODES[c["dtype"]]
    if c["op"] == "norm":
        h, ch = c["heads"], c["channels"]
        state["desc"] = odla.RmsNormDesc(dtype=dt, weight_dtype=CODES[c["weight"]], rows=c["rows"], heads=h, channels=ch, quant=EIGHT[c["eight"]], group=c["group"] if c["scales"] == "own" else 0,
                                         epsilon=EPSILON, weight_offset=0.0, x_row=state["x"].stride(0), x_head=ch, residual_row=h * ch, residual_head=ch, sum_row=h * ch, sum_head=ch, y_row=h * ch,
                                         y_head=ch, quant_row=h * ch, quant_head=ch)
        if c["eight"] == "s8":
            state["values"] = torch.empty(state["eight"].shape, dtype=torch.float16, device="cuda")
    elif c["op"] == "log_probs":
        state["desc"] = odla.LogProbsDesc(dtype=dt, rows=c["rows"], vocab=c["vocab"], given=c["given"], top=c["top"], row=c["vocab"])
    else:
        h, kh, d, page = c["heads"], c["kv_heads"], c["channels"], c["page"]
        head, token = (d, kh * d) if c["token_major"] else (page * d, d)
        state["cache"] = odla.PagedCache(dtype=dt, pages=state["key_cache"].shape[0], page_size=page, heads=kh, channels=d, page=page * kh * d, head=head, token=token)
        state["desc"] = odla.ChunkAttentionDesc(batch=c["batch"], tokens=state["q"].shape[0], heads=h, prefix_length=c["prefix"], table_width=state["table"].shape[1], scale=1 / math.sqrt(d),
                                                q_token=h * d, q_head=d, y_token=h * d, y_head=d)


def _own(s, c):
    if "lib" not in s:
        _bind(s)
    lib, ref, stream = s["lib"], ctypes.byref, torch.cuda.current_stream().cuda_stream

    def p(name):
        return s[name].data_ptr() if name in s else None
    if c["op"] == "norm":
        rc = lib.b200_rms_norm(ref(s["desc"]), p("x"), p("residual"), p("weight"), p("sum"), p("y"), p("eight"), p("scales"), stream)
        out = [s[n] for n in ("sum", "y") if n in s] + ([s["scales"]] if c["scales"] == "own" else [])
        if c["eight"] == "e4m3":
            out.append(s["eight"])
        elif c["eight"] == "s8":                         # what 8 bits stand for
            scales = s["scales"][..., None] if c["scales"] == "own" else s["scales"]
            groups = (-1, c["group"])
            out.append(torch.mul(s["eight"].unflatten(-1, groups), scales, out=s["values"].unflatten(-1, groups)).flatten(-2))
    elif c["op"] == "log_probs":
        out = [s["given"], s["entropy"], s["top_tokens"], s["top"]]
        rc = lib.b200_log_probs(ref(s["desc"]), p("logits"), p("temperature"), p("tokens"), p("given"), p("entropy"), p("top_tokens"), p("top"), stream)
    else:
        out = s["y"]
        rc = lib.b200_chunk_attention(ref(s["cache"]), p("key_cache"), p("value_cache"), ref(s["desc"]), p("q"), p("starts"), p("prefix_pages"), p("table"), p("lengths"), p("y"), stream)
    if rc:
        raise RuntimeError("%s failed with %d" % (c["op"], rc))
    return out


def run(state):
    c = state["case"]
    if own:
        return _own(state, c)
    return {"norm": _plain_norm, "chunk": _plain_chunk, "log_probs": _plain_log_probs}[c["op"]](state, c)


# ------------------------------------------------------------------- the definition ----
def _exact_norm(s, c):
    x = s["x"].narrow(1, 0, c["heads"]).double()
    out = []
    if c["residual"]:
        h = x + s["residual"].double()
        out.append(h)
        x = h.to(s["x"].dtype).double()                  # (the norm is that of the sum as it is stored)
    y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["channels"] + EPSILON) * s["weight"].double()
    if c["plain_out"]:
        out.append(y)
    if c["eight"] == "none":
        return out
    most = LARGEST[c["eight"]]
    z = y.reshape(c["rows"], c["heads"], -1, c["group"])
    if c["scales"] == "own":
        scale = z.abs().max(-1).values / most
        out.append(scale)
    else:
        scale = s["scales"].double().reshape(1, 1, 1)
    scale = scale.unsqueeze(-1)
    q = z / scale.clamp(min=1e-300)
    if c["eight"] == "s8":
        q = q.round().clamp(-128, 127) * scale
    else:                                                # e4m3: three bits behind the point, of steps of 2^-9 at least
        q = q.clamp(-most, most)
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
        q = (q / step).round() * step
    out.append(q.reshape(y.shape))
    return out


def _exact_chunk(s, c):
    h, kh, d, page = c["heads"], c["kv_heads"], c["channels"], c["page"]
    kc, vc = ((x if c["token_major"] else x.transpose(1, 2)).reshape(-1, kh, d) for x in (s["key_cache"], s["value_cache"]))      # one row per slot

    def slots(pages, n):
        i = torch.arange(n, device="cuda")
        return pages.long()[i // page] * page + i % page
    shared = slots(s["prefix_pages"], c["prefix"])
    out = s["y"].double()
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    for b, n in enumerate(lengths):
        first, count = starts[b], starts[b + 1] - starts[b]
        if not count:
            continue
        at = torch.cat([shared, slots(s["table"][b], n)])
        k, v = kc[at].double(), vc[at].double()
        for lo in range(0, count, 1024):
            rows = range(lo, min(count, lo + 1024))
            sees = torch.tensor([c["prefix"] + n - count + j + 1 for j in rows], device="cuda")
            hidden = torch.arange(len(at), device="cuda")[None, :] >= sees[:, None]
            for j in range(h):
                e = s["q"][first + rows.start:first + rows.stop, j].double() @ k[:, j // (h // kh)].T / math.sqrt(d)
                out[first + rows.start:first + rows.stop, j] = torch.softmax(e.masked_fill(hidden, -math.inf), dim=-1) @ v[:, j // (h // kh)]
    return out


def _exact_log_probs(s, c):
    z = s["logits"].double()
    if c["scaled"]:
        z = z / s["temperature"].double()[:, None]
    logp = torch.log_softmax(z, dim=-1)
    entropy = torch.special.entr(logp.exp()).sum(-1)
    rows = torch.arange(c["rows"], device="cuda")[:, None]
    given = logp[rows, s["tokens"].long()]
    given[s["tokens"] < 0] = -math.inf
    # the largest one, struck out, over and over: argmax takes the first of equals
    left, tokens = s["logits"].double(), []
    for _ in range(c["top"]):
        i = (left == left.max(-1, keepdim=True).values).to(torch.uint8).argmax(-1)
        tokens.append(torch.where(left[rows[:, 0], i] > -math.inf, i, -1))
        left[rows[:, 0], i] = -math.inf
    tokens = torch.stack(tokens, 1) if tokens else torch.empty((c["rows"], 0), dtype=torch.int64, device="cuda")
    top = torch.where(tokens >= 0, logp.gather(1, tokens.clamp(min=0)), -math.inf)
    return [given, entropy, tokens.to(torch.int32), top]


def exact(case, seed):
    return {"norm": _exact_norm, "chunk": _exact_chunk, "log_probs": _exact_log_probs}[case["op"]](prepare(case, seed), case)
