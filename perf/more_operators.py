"""Timed cases of the paged cache of keys and values, through the Python binding
of the C ABI.

Kinds of case:

  append     raw projections of new tokens: queries and keys normalised per head
             and rotated by one to three position axes, keys and values written
             to the pages of their requests
  attention  gated attention of each request's new tokens, one or a chunk of
             them, over its paged keys, all of them or a window behind the first
             few (sinks)
  weights    what those tokens attend to, added up per cached key
  evict      the keys of largest accumulated weight kept, moved to other pages

Widths come from the layer shapes of workloads.block_config (16 query and 2 key
heads x 256, rotary on 64 features, three position axes of 11, 11 and 10 pairs)
and from the shapes of the attention tests.
"""
import importlib
import math
import random

import torch

own = False

DEV = "cuda"
DT = {"f16": torch.float16, "f32": torch.float32}
BYTES = {"f16": 2, "f32": 4}
THETA = 10000000.0
EPS = 1e-6
SECTIONS = {1: [1.0], 2: [0.5, 0.5], 3: [11 / 32, 11 / 32, 10 / 32]}


def listed():
    layer = {"heads": 16, "kv_heads": 2, "d": 256}
    return [
        # one request's next token enters the cache: the smallest call
        {"name": "append_1", "kind": "append", "dtype": "f16", "requests": 1, "tokens": 1, "cached": 900, "uneven": 1,
         "page": 64, "rot": 64, "axes": 1, "far": 0, **layer},
        # prompts of eight requests with images: positions of three axes
        {"name": "append_8_1024", "kind": "append", "dtype": "f16", "requests": 8, "tokens": 1024, "cached": 512,
         "uneven": 2, "page": 64, "rot": 64, "axes": 3, "far": 0, **layer},
        # one request's next token, a short conversation: latency counts
        {"name": "paged_1_700", "kind": "attention", "dtype": "f16", "requests": 1, "tokens": 1, "cached": 700,
         "uneven": 3, "page": 64, "window": 0, "sinks": 0, **layer},
        # a full batch of answers in long, uneven conversations
        {"name": "paged_64_16384", "kind": "attention", "dtype": "f16", "requests": 64, "tokens": 1, "cached": 16384,
         "uneven": 4, "page": 64, "window": 0, "sinks": 0, **layer},
        # a chunk of a long document's prompt over what is cached of it
        {"name": "paged_chunk_1024", "kind": "attention", "dtype": "f16", "requests": 1, "tokens": 1024,
         "cached": 16384, "uneven": 5, "page": 64, "window": 0, "sinks": 0, **layer},
        # chunks of uneven requests in a stream without end: a window and four sinks
        {"name": "paged_window_4", "kind": "attention", "dtype": "f16", "requests": 4, "tokens": 1500,
         "cached": 9000, "uneven": 6, "page": 32, "window": 1024, "sinks": 4, **layer},
        # the f32 profile: a few tokens each of a few requests, small pages
        {"name": "paged_f32_5", "kind": "attention", "dtype": "f32", "requests": 5, "tokens": 3, "cached": 1333,
         "uneven": 7, "page": 16, "window": 0, "sinks": 0, **layer},
        # the step of a batch whose caches are to be cut: weights of the newest token
        {"name": "weights_32_8192", "kind": "weights", "dtype": "f16", "requests": 32, "tokens": 1, "cached": 8192,
         "uneven": 8, "page": 64, "window": 0, "sinks": 0, **layer},
        # the last tokens of a prompt look back on it
        {"name": "weights_chunk_333", "kind": "weights", "dtype": "f16", "requests": 1, "tokens": 333, "cached": 4096,
         "uneven": 9, "page": 64, "window": 0, "sinks": 0, **layer},
        # one short conversation cut to half, f32 profile
        {"name": "evict_f32_1", "kind": "evict", "dtype": "f32", "requests": 1, "cached": 1500, "uneven": 10,
         "page": 64, "budget": 700, "sinks": 4, "recent": 64, **layer},
        # a batch of long conversations cut to a quarter
        {"name": "evict_16_16384", "kind": "evict", "dtype": "f16", "requests": 16, "cached": 16384, "uneven": 11,
         "page": 64, "budget": 4096, "sinks": 4, "recent": 512, **layer},
    ]


def _log(rng, lo, hi):
    """An integer spread evenly over the logarithm of lo..hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "attention", "weights", "evict"])
    kv_heads = rng.choice([2, 2, 1, 4])
    case = {"kind": kind, "dtype": rng.choice(["f16", "f16", "f32"]), "uneven": rng.randint(12, 10 ** 6),
            "page": rng.choice([64, 64, 16, 32, 128]), "d": rng.choice([256, 256, 128, 64, 72]),
            "kv_heads": kv_heads, "heads": kv_heads * min(16 // kv_heads, rng.choice([8, 4, 1, 3]))}
    if kind == "evict":
        n = _log(rng, 1, 16)
        cached = _log(rng, 32, 16384 if case["dtype"] == "f16" else 8192)
        budget = max(8, int(cached * rng.uniform(0.1, 0.8)))
        return {**case, "requests": n, "cached": cached, "budget": budget, "sinks": rng.choice([0, 4, 1]),
                "recent": rng.randint(0, budget // 4)}
    if kind == "append":
        n = _log(rng, 1, 32)
        rot = min(case["d"], rng.choice([64, 64, 32, 256])) // 8 * 8
        return {**case, "requests": n, "tokens": _log(rng, 1, 8192 // n), "cached": _log(rng, 1, 4096), "rot": rot,
                "axes": rng.choice([1, 3, 2]), "far": rng.choice([0, 0, rng.randint(1, 10 ** 6)])}
    # single tokens of many requests, a few tokens each, or chunks of few requests
    tokens, n = rng.choice([(1, _log(rng, 1, 64)), (_log(rng, 2, 12), _log(rng, 1, 32)),
                            (_log(rng, 13, 1024), _log(rng, 1, 6))])
    # as much as a chunk of 1,024 tokens behind 16,384 at most (a sixteenth of it in f32)
    most = (1 << 24) // (1 if case["dtype"] == "f16" else 16) // (n * tokens)
    cached = _log(rng, 1, max(2, min(16384, most, (1 << 21) // (n * kv_heads))))
    window = rng.choice([0, 0, _log(rng, 1, 2048)])
    return {**case, "requests": n, "tokens": tokens, "cached": cached, "window": window,
            "sinks": rng.choice([0, 4, 64]) if window else 0}


# --------------------------------------------------------------------------- sizes that follow from a case
def _lengths(case):
    """(new tokens, cached tokens with them) of each request; one of each case has the most."""
    rng = random.Random(case["uneven"])
    n, tokens, cached = case["requests"], case.get("tokens", 0), case["cached"]
    new = [tokens if i == 0 or tokens < 2 else rng.randint((tokens + 1) // 2, tokens) for i in range(n)]
    old = [cached if i == 0 else rng.randint(cached // 8, cached) for i in range(n)]
    return new, [a + b for a, b in zip(new, old)]


def _axis_of(case):
    """The axis of each rotary pair: dealt in turn while the shorter sections last."""
    half = case["rot"] // 2
    left = [int(round(half * x)) for x in SECTIONS[case["axes"]][1:]]
    out = [0] * half
    for axis, count in enumerate(left, 1):
        for i in range(count):
            at = axis + i * case["axes"]
            if at < half:
                out[at] = axis
    return out


def _seen(case, p):
    """How many of the keys 0 .. p a query at p sees."""
    if not case["window"]:
        return p + 1
    return min(p + 1, case["window"] + min(case["sinks"], max(0, p + 1 - case["window"])))


# --------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    if dtype == torch.float32:
        return torch.randn(shape, generator=g, device=DEV) * std
    return torch.randn(shape, generator=g, device=DEV, dtype=dtype).mul_(std)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _table(g, case, lens, extra=0):
    """Pages of each request, scattered over the pool; what a request does not reach names no page."""
    counts = [-(-x // case["page"]) for x in lens]
    width, total = max(counts) + extra, sum(counts)
    order = torch.randperm(total + extra, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, c in enumerate(counts):
        table[s, :c] = order[at:at + c]
        at += c
    return table, total + extra


def _pool(g, case, pages):
    kvh, page, d, dt = case["kv_heads"], case["page"], case["d"], DT[case["dtype"]]
    return _randn(g, pages, kvh, page, d, dtype=dt), _randn(g, pages, kvh, d, page, dtype=dt)


def _positions(case, new, lens):
    """Positions of three axes: text counts on all of them, a picture of w columns
    stands still on the first and counts rows and columns on the others."""
    rng = random.Random(case["uneven"] + 1)
    rows = []
    for n, m in zip(new, lens):
        first, w = m - n + case["far"], rng.randint(3, 40)
        inside = (n // 4, n // 4 + n // 2)
        for i in range(n):
            if inside[0] <= i < inside[1]:
                j = i - inside[0]
                rows.append([first + inside[0], first + inside[0] + j // w, first + inside[0] + j % w])
            else:
                rows.append([first + i] * 3)
    return _ints(rows).t()[:case["axes"]].contiguous()


def prepare(case, seed):
    g = _gen(seed)
    dt, d, heads, kvh, page = DT[case["dtype"]], case["d"], case["heads"], case["kv_heads"], case["page"]
    new, lens = _lengths(case)
    table, pages = _table(g, case, lens, 3)
    k, vt = _pool(g, case, pages)
    s = {"case": case, "k": k, "vt": vt, "table": table, "len": _ints(lens)}
    if own:
        clef = importlib.import_module("clef-rs_amd.clef_hip")
        s["cache"] = clef.PagedCache(k, vt)
    if case["kind"] == "evict":
        kept = [min(x, case["budget"]) for x in lens]
        s["to_table"], to_pages = _table(g, case, kept, 1)
        s["to_k"], s["to_vt"] = (torch.zeros(to_pages, *x.shape[1:], dtype=dt, device=DEV) for x in (k, vt))
        # heavy-tailed sums, and keys that nothing has looked at
        s["scores"] = torch.exp(_randn(g, pages, kvh, page, std=3.0))
        s["scores"] *= torch.rand((pages, kvh, page), generator=g, device=DEV) > 0.1
        s["to_scores"] = torch.zeros((to_pages, kvh, page), device=DEV)
        if own:
            s["to"] = clef.PagedCache(s["to_k"], s["to_vt"])
        return s
    t = sum(new)
    s["cu"] = _ints([sum(new[:i]) for i in range(len(new) + 1)])
    if case["kind"] == "append":
        # one packed projection: [query | gate] of each head, keys, values
        s["x"] = _randn(g, t, (2 * heads + 2 * kvh) * d, dtype=dt)
        s["q_norm"], s["k_norm"] = 1.0 + _randn(g, d, std=0.1), 1.0 + _randn(g, d, std=0.1)
        s["positions"] = _positions(case, new, lens)
        s["axis_of"] = _axis_of(case)
        return s
    s["q"] = _randn(g, heads, t, d, dtype=dt)
    if case["kind"] == "attention":
        s["gate"] = _randn(g, t, heads, d, dtype=dt)
        return s
    # sums of a few earlier calls like this one
    s["scores"] = torch.exp(_randn(g, pages, kvh, page)) * (case["tokens"] * heads / kvh / case["cached"])
    # the pool that the new sums go to, so that a draft can be taken back
    s["new_scores"] = s["scores"].clone()
    s["lse"] = _log_sums(s)
    return s


def _log_sums(s):
    """What the attention of the same tokens leaves: the logarithm of each row's sum."""
    case = s["case"]
    out = torch.empty((s["q"].shape[1], case["heads"]), device=DEV)
    rep = case["heads"] // case["kv_heads"]
    new, lens = _lengths(case)
    t = 0
    for r, (n, m) in enumerate(zip(new, lens)):
        pages = s["table"][r, :-(-m // case["page"])].long()
        k = s["k"][pages].transpose(0, 1).reshape(case["kv_heads"], 1, -1, case["d"])[:, :, :m].double()
        p = torch.arange(m - n, m, device=DEV)[:, None]
        j = torch.arange(m, device=DEV)[None, :]
        seen = (j <= p) & ((j < case["sinks"]) | (j > p - case["window"])) if case["window"] else j <= p
        q = s["q"][:, t:t + n].view(case["kv_heads"], rep, n, case["d"]).double() / math.sqrt(case["d"])
        for h in range(rep):
            w = torch.matmul(q[:, h], k[:, 0].transpose(1, 2)).masked_fill(~seen, float("-inf"))
            out[t:t + n, h::rep] = torch.logsumexp(w, -1).t().float()
        t += n
    return out


# --------------------------------------------------------------------------- one pass
def run(s):
    return (_run_own if own else _run_plain)(s)


def _projections(s):
    """Views of the packed projection: q, k, v [T, heads, d]."""
    case, x = s["case"], s["x"]
    t, heads, kvh, d = x.shape[0], case["heads"], case["kv_heads"], case["d"]
    q = x[:, :2 * heads * d].view(t, heads, 2 * d)[:, :, :d]
    k = x[:, 2 * heads * d:(2 * heads + kvh) * d].view(t, kvh, d)
    return q, k, x[:, (2 * heads + kvh) * d:].view(t, kvh, d)


def _run_own(s):
    case, cache = s["case"], s["cache"]
    if case["kind"] == "append":
        q, k, v = _projections(s)
        q = cache.append(q, k, v, s["q_norm"], s["k_norm"], s["cu"], s["len"], s["table"], case["rot"], THETA,
                         positions=s["positions"], axis_of=s["axis_of"], eps=EPS)
        return {"q": q, "k": s["k"], "vt": s["vt"]}
    if case["kind"] == "attention":
        return cache.attention_gated(s["q"], s["gate"], s["cu"], s["len"], s["table"], window=case["window"],
                                     sinks=case["sinks"])
    if case["kind"] == "weights":
        return cache.add_weights(s["q"], s["lse"], s["cu"], s["len"], s["table"], s["scores"],
                                 new_scores=s["new_scores"], window=case["window"], sinks=case["sinks"])
    lens, keep = cache.evict(s["scores"], s["len"], s["table"], case["budget"], s["to"], s["to_table"],
                             s["to_scores"], sinks=case["sinks"], recent=case["recent"])
    return {"lens": lens, "keep": keep, "k": s["to_k"], "vt": s["to_vt"], "scores": s["to_scores"]}


def _run_plain(s):
    return {"append": _plain_append, "attention": _plain_attention, "weights": _plain_weights,
            "evict": _plain_evict}[s["case"]["kind"]](s)


def _tokens(s):
    """(request, key index) of each packed token."""
    cu, t = s["cu"].long(), s["x"].shape[0] if "x" in s else s["q"].shape[1]
    at = torch.arange(t, device=DEV)
    seq = torch.searchsorted(cu[1:], at, right=True)
    return seq, s["len"].long()[seq] - (cu[seq + 1] - at)


def _plain_append(s):
    case, dt = s["case"], s["x"].dtype
    half = case["rot"] // 2
    seq, index = _tokens(s)
    axis = torch.tensor(s["axis_of"], device=DEV)
    freq = THETA ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
    angle = s["positions"].double()[axis].t() * freq  # [T, pairs]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turned(x, w):
        x = x.float()
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1).to(dt)

    q, k, v = _projections(s)
    page, slot = s["table"].long()[seq, index // case["page"]], index % case["page"]
    s["k"][page, :, slot] = turned(k, s["k_norm"])
    s["vt"][page, :, :, slot] = v
    return {"q": turned(q, s["q_norm"]).transpose(0, 1).contiguous(), "k": s["k"], "vt": s["vt"]}


def _padded(s):
    """Queries padded to the longest request's, keys to the table's width: (q [n, kvh,
    rep, m, d], keys [n, kvh, 1, j, d], seen [n, 1, 1, m, j], the packed tokens' places)."""
    case = s["case"]
    n, t = case["requests"], s["q"].shape[1]
    seq, index = _tokens(s)
    new = (s["cu"][1:] - s["cu"][:-1]).long()
    most, rep = case["tokens"], case["heads"] // case["kv_heads"]
    row = torch.arange(t, device=DEV) - s["cu"].long()[seq]
    q = torch.zeros((n, most, case["heads"], case["d"]), device=DEV)
    q[seq, row] = s["q"].float().transpose(0, 1)
    q = q.view(n, most, case["kv_heads"], rep, case["d"]).permute(0, 2, 3, 1, 4)
    keys = s["k"][s["table"].long().clamp(min=0)].float().transpose(1, 2).reshape(n, case["kv_heads"], 1, -1, case["d"])
    j = torch.arange(keys.shape[3], device=DEV)
    p = (s["len"].long() - new)[:, None] + torch.arange(most, device=DEV)
    seen = (j <= p[..., None]) & (torch.arange(most, device=DEV) < new[:, None])[..., None]
    if case["window"]:
        seen &= (j < case["sinks"]) | (j > p[..., None] - case["window"])
    return q, keys, seen[:, None, None], (seq, row)


def _plain_attention(s):
    case, dt = s["case"], s["q"].dtype
    q, keys, seen, (seq, row) = _padded(s)
    values = s["vt"][s["table"].long().clamp(min=0)].float().permute(0, 2, 3, 1, 4)
    values = values.reshape(case["requests"], case["kv_heads"], 1, case["d"], -1)
    scores = torch.where(seen, q @ keys.transpose(-1, -2) / math.sqrt(case["d"]), float("-inf"))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = e.sum(-1, keepdim=True)
    out = (e @ values.transpose(-1, -2)) / torch.where(total == 0, 1.0, total)
    out = out.permute(0, 3, 1, 2, 4).reshape(case["requests"], -1, case["heads"], case["d"])[seq, row]
    return (out / (1.0 + torch.exp(-s["gate"].float()))).to(dt).reshape(out.shape[0], -1)


def _plain_weights(s):
    case = s["case"]
    q, keys, seen, (seq, row) = _padded(s)
    n, kvh = case["requests"], case["kv_heads"]
    lse = torch.zeros((n, case["tokens"], case["heads"]), device=DEV)
    lse[seq, row] = s["lse"]
    lse = lse.view(n, -1, kvh, case["heads"] // kvh).permute(0, 2, 3, 1)[..., None]
    scores = q @ keys.transpose(-1, -2) / math.sqrt(case["d"])
    total = torch.where(seen, torch.exp(scores - lse), 0.0).sum((2, 3))  # [n, kvh, keys]
    j = torch.arange(total.shape[2], device=DEV)
    new = (s["cu"][1:] - s["cu"][:-1]).long()
    length = s["len"].long()[:, None]
    page = s["table"].long()[:, j // case["page"]]
    r, at = torch.nonzero((j < length), as_tuple=True)
    before = torch.where(at < length[r, 0] - new[r], 1.0, 0.0)[:, None]
    where = (page[r, at], slice(None), at % case["page"])
    s["new_scores"][where] = s["scores"][where] * before + total[r, :, at]
    return s["new_scores"]


def _plain_evict(s):
    case = s["case"]
    n, kvh, size, budget = case["requests"], case["kv_heads"], case["page"], case["budget"]
    table, to = s["table"].long().clamp(min=0), s["to_table"].long()
    flat = s["scores"][table].transpose(1, 2).reshape(n, kvh, -1)
    j = torch.arange(flat.shape[2], device=DEV)
    length = s["len"].long()[:, None, None]
    always = (j < case["sinks"]) | (j >= length - case["recent"])
    rank = torch.where(always, float("inf"), flat)
    rank = torch.where(j < length, rank, float("-inf"))
    lens = s["len"].clamp(max=budget)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    if order.shape[2] < budget:
        order = torch.nn.functional.pad(order, (0, budget - order.shape[2]), value=flat.shape[2])
    slot = torch.arange(budget, device=DEV)
    kept = slot < lens[:, None, None]
    order = torch.sort(torch.where(kept, order, flat.shape[2]), dim=-1).values
    keep = torch.where(kept, order, -1).to(torch.int32)
    r, h, i = torch.nonzero(keep >= 0, as_tuple=True)
    at = order[r, h, i]
    a, b = (table[r, at // size], h, at % size), (to[r, i // size], h, i % size)
    s["to_k"][b] = s["k"][a]
    s["to_scores"][b] = s["scores"][a]
    s["to_vt"][b[0], h, :, b[2]] = s["vt"][a[0], h, :, a[2]]
    return {"lens": lens, "keep": keep, "k": s["to_k"], "vt": s["to_vt"], "scores": s["to_scores"]}


# --------------------------------------------------------------------------- least work
def work(case):
    e = BYTES[case["dtype"]]
    heads, kvh, d = case["heads"], case["kv_heads"], case["d"]
    new, lens = _lengths(case)
    t = sum(new)
    if case["kind"] == "append":
        rows = heads + 2 * kvh
        return {"bytes": 2 * e * t * rows * d + 4 * t * case["axes"], "flops": 6 * t * (heads + kvh) * d}
    if case["kind"] == "evict":
        kept = sum(min(x, case["budget"]) for x in lens)
        return {"bytes": 4 * kvh * sum(lens) + kept * kvh * (4 * d * e + 4 + 4 + 4), "flops": kvh * sum(lens)}
    pairs = keys = 0
    for n, m in zip(new, lens):
        pairs += sum(_seen(case, p) for p in range(m - n, m))
        first = max(0, m - n - case["window"] + 1) if case["window"] else 0
        keys += m - first + min(case["sinks"], first)
    if case["kind"] == "attention":
        return {"bytes": e * (3 * t * heads * d + 2 * keys * kvh * d), "flops": 4 * heads * d * pairs}
    return {"bytes": e * (t * heads * d + keys * kvh * d) + 4 * t * heads + 8 * kvh * sum(lens),
            "flops": 2 * heads * d * pairs}


# --------------------------------------------------------------------------- 64-bit results
def exact(case, seed):
    s = prepare(case, seed)
    new, lens = _lengths(case)
    heads, kvh, d, size = case["heads"], case["kv_heads"], case["d"], case["page"]
    rep = heads // kvh
    tables = s["table"].tolist()

    def cached(pool, r, count):
        """Request r's first rows of a pool [pages, kvh, page, ...]: [kvh, count, ...]."""
        used = tables[r][:-(-count // size)]
        return torch.cat([pool[x] for x in used], 1)[:, :count]

    if case["kind"] == "append":
        half = case["rot"] // 2
        q, k, v = _projections(s)
        out, pk, pv = q.double().transpose(0, 1).clone(), s["k"].double(), s["vt"].double()
        places = s["positions"].tolist()
        angles = torch.tensor([[places[a][i] * THETA ** (-2.0 * p / case["rot"]) for p, a in enumerate(s["axis_of"])]
                               for i in range(q.shape[0])], dtype=torch.float64, device=DEV)
        turn = torch.complex(torch.cos(angles), torch.sin(angles))[:, None]

        def rotated(x, w):
            x = x.double() * torch.rsqrt(x.double().pow(2).sum(-1, keepdim=True) / d + EPS) * w.double()
            z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
            x[..., :half], x[..., half:2 * half] = z.real, z.imag
            return x

        out = rotated(q, s["q_norm"]).transpose(0, 1)
        keys = rotated(k, s["k_norm"])
        t = 0
        for r, (n, m) in enumerate(zip(new, lens)):
            i = 0
            while i < n:
                at = m - n + i
                run_ = min(n - i, size - at % size)
                page, first = tables[r][at // size], at % size
                pk[page, :, first:first + run_] = keys[t + i:t + i + run_].transpose(0, 1)
                pv[page, :, :, first:first + run_] = v[t + i:t + i + run_].double().permute(1, 2, 0)
                i += run_
            t += n
        return {"q": out, "k": pk, "vt": pv}

    if case["kind"] == "evict":
        pk, pv, ps = s["to_k"].double(), s["to_vt"].double(), s["to_scores"].double()
        to = s["to_table"].tolist()
        chosen = torch.full((len(lens), kvh, case["budget"]), -1, dtype=torch.int32)
        for r, m in enumerate(lens):
            sums, keys = cached(s["scores"], r, m), cached(s["k"], r, m).double()
            weight = sums.tolist()
            values = cached(s["vt"].transpose(2, 3), r, m).double()
            most = min(m, case["budget"])
            for h in range(kvh):
                fixed = set(range(min(case["sinks"], m))) | set(range(max(0, m - case["recent"]), m))
                rest = sorted((j for j in range(m) if j not in fixed), key=lambda j: (-weight[h][j], j))
                keep = range(m) if m <= most else sorted(fixed | set(rest[:most - len(fixed)]))
                chosen[r, h, :most] = torch.tensor(list(keep))
                at = torch.tensor(list(keep), device=DEV)
                for i in range(0, most, size):
                    some, count = at[i:i + size], min(size, most - i)
                    pk[to[r][i // size], h, :count] = keys[h, some]
                    pv[to[r][i // size], h, :, :count] = values[h, some].t()
                    ps[to[r][i // size], h, :count] = sums[h, some].double()
        return {"lens": _ints([min(m, case["budget"]) for m in lens]), "keep": chosen.to(DEV), "k": pk, "vt": pv, "scores": ps}

    if sum(n * m for n, m in zip(new, lens)) * heads > 1 << 33:
        return None
    out = torch.empty((sum(new), heads, d), dtype=torch.float64, device=DEV)
    sums = s["new_scores"].double() if case["kind"] == "weights" else None
    t = 0
    for r, (n, m) in enumerate(zip(new, lens)):
        keys = cached(s["k"], r, m).double()
        values = cached(s["vt"].transpose(2, 3), r, m).double() if sums is None else None
        total = torch.zeros((kvh, m), dtype=torch.float64, device=DEV)
        step = max(1, (1 << 27) // (rep * m))
        for i0 in range(0, n, step):
            rows = range(i0, min(n, i0 + step))
            hide = torch.ones((len(rows), m), dtype=torch.bool, device=DEV)
            for x, i in enumerate(rows):
                p = m - n + i
                if not case["window"]:
                    hide[x, :p + 1] = False
                else:
                    hide[x, max(0, p + 1 - case["window"]):p + 1] = False
                    hide[x, :min(case["sinks"], p + 1)] = False
            for h in range(kvh):
                q = s["q"][h * rep:(h + 1) * rep, t + i0:t + i0 + len(rows)].double()
                z = (q.reshape(-1, d) @ keys[h].t()).view(rep, len(rows), m) / math.sqrt(d)
                if sums is None:
                    w = torch.softmax(z.masked_fill(hide, float("-inf")), -1)
                    y = (w.reshape(-1, m) @ values[h]).view(rep, len(rows), d).transpose(0, 1)
                    out[t + i0:t + i0 + len(rows), h * rep:(h + 1) * rep] = y
                else:
                    lse = s["lse"][t + i0:t + i0 + len(rows), h * rep:(h + 1) * rep].double().t()[..., None]
                    total[h] += torch.exp(z - lse).masked_fill(hide, 0.0).sum((0, 1))
        if sums is not None:
            before = cached(s["scores"], r, m).double()
            before[:, m - n:] = 0.0
            total += before
            for i in range(0, m, size):
                sums[tables[r][i // size], :, :min(size, m - i)] = total[:, i:i + size]
        t += n
    if sums is not None:
        return sums
    return (out * torch.sigmoid(s["gate"].double())).reshape(out.shape[0], -1)
