"""Timed cases of the linear-attention and shared-prefix operators, through the
Python binding of the C ABI.

Kinds of case:

  linear       linear attention with one decay per head over a prompt, or over
               a ragged batch of prompts (chunked form, final states out)
  linear_step  the same recurrence for one token of each of a batch of requests
  delta_step   the gated-DeltaNet recurrence for one token of each request
  shared       gated attention of a batch of requests, one to a few tokens
               each, behind one shared prefix and each request's own keys

Widths come from the layer shapes of workloads.block_config (DeltaNet 16 key
and 32 value heads x 128, attention 16 query and 2 key heads x 256) and from
the shapes of the scan and attention tests.
"""
import importlib
import math
import random

import torch

own = False

DEV = "cuda"
DT = {"f16": torch.float16, "f32": torch.float32}
BYTES = {"f16": 2, "f32": 4}


def listed():
    return [
        # a question of a few words, alone: the smallest prompt, where latency counts
        {"name": "linear_33", "kind": "linear", "dtype": "f16", "tokens": 33, "requests": 1, "uneven": 0,
         "hk": 4, "hv": 4, "dk": 64, "dv": 64, "initial": "none", "decay": "slopes"},
        # a batch of uneven requests resumed from one shared prefix state
        {"name": "linear_ragged_8", "kind": "linear", "dtype": "f16", "tokens": 5003, "requests": 8, "uneven": 1,
         "hk": 16, "hv": 32, "dk": 128, "dv": 128, "initial": "shared", "decay": "slopes"},
        # the f32 profile (parity and evaluation), an odd length resumed from a state
        {"name": "linear_f32_1001", "kind": "linear", "dtype": "f32", "tokens": 1001, "requests": 1, "uneven": 0,
         "hk": 16, "hv": 32, "dk": 128, "dv": 128, "initial": "shared", "decay": "slopes"},
        # a long document in one pass
        {"name": "linear_16384", "kind": "linear", "dtype": "f16", "tokens": 16384, "requests": 1, "uneven": 0,
         "hk": 16, "hv": 32, "dk": 128, "dv": 128, "initial": "none", "decay": "slopes"},
        # one request's next token
        {"name": "linear_step_1", "kind": "linear_step", "dtype": "f16", "rows": 1, "slots": 1, "padded": 0,
         "hk": 16, "hv": 32, "dk": 128, "dv": 128, "decay": "slopes"},
        # a batch's next tokens, states in a pool, some rows of the batch empty
        {"name": "linear_step_64", "kind": "linear_step", "dtype": "f16", "rows": 64, "slots": 96, "padded": 5,
         "hk": 16, "hv": 32, "dk": 128, "dv": 128, "decay": "slopes"},
        # a few requests of the f32 profile
        {"name": "delta_step_f32_3", "kind": "delta_step", "dtype": "f32", "rows": 3, "slots": 3, "padded": 0,
         "hk": 16, "hv": 32, "dk": 128, "dv": 128},
        # the next token of a full batch of the hybrid layer's shape
        {"name": "delta_step_128", "kind": "delta_step", "dtype": "f16", "rows": 128, "slots": 128, "padded": 0,
         "hk": 16, "hv": 32, "dk": 128, "dv": 128},
        # two requests behind a short prefix: the smallest call
        {"name": "shared_2_512", "kind": "shared", "dtype": "f16", "requests": 2, "tokens": 1, "uneven": 2,
         "prefix": 512, "room": 64, "heads": 16, "kv_heads": 2, "d": 256},
        # a batch of 32 requests in the middle of their answers
        {"name": "shared_32_4096", "kind": "shared", "dtype": "f16", "requests": 32, "tokens": 1, "uneven": 3,
         "prefix": 4096, "room": 256, "heads": 16, "kv_heads": 2, "d": 256},
        # the f32 profile, up to five tokens a request, an odd prefix, caches at odd places
        {"name": "shared_f32_7_777", "kind": "shared", "dtype": "f32", "requests": 7, "tokens": 5, "uneven": 4,
         "prefix": 777, "room": 151, "heads": 16, "kv_heads": 2, "d": 256},
        # a large batch behind a long document
        {"name": "shared_128_32768", "kind": "shared", "dtype": "f16", "requests": 128, "tokens": 1, "uneven": 5,
         "prefix": 32768, "room": 256, "heads": 16, "kv_heads": 2, "d": 256},
    ]


def _log(rng, lo, hi):
    """An integer spread evenly over the logarithm of lo..hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(16, 32), (16, 32), (4, 4), (2, 6), (8, 8), (1, 5)]
WIDTHS = [(128, 128), (128, 128), (64, 64), (64, 128), (128, 13), (100, 72), (40, 24)]


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear_step", "delta_step", "shared", "shared"])
    dtype = rng.choice(["f16", "f16", "f32"])
    if kind == "shared":
        d = rng.choice([256, 256, 128, 64, 72])
        kv_heads = rng.choice([2, 2, 1, 4])
        heads = kv_heads * min(16 // kv_heads, rng.choice([8, 4, 1, 3]))
        tokens = rng.choice([1, 1, 1, rng.randint(2, 8)])
        requests = _log(rng, 1, 128 if tokens == 1 else 128 // tokens)
        return {"kind": kind, "dtype": dtype, "requests": requests, "tokens": tokens, "uneven": rng.randint(6, 10 ** 6),
                "prefix": _log(rng, 8, 32768 if dtype == "f16" else 8192), "room": _log(rng, 8, 256),
                "heads": heads, "kv_heads": kv_heads, "d": d}
    hk, hv = rng.choice(HEADS)
    dk, dv = rng.choice(WIDTHS)
    decay = rng.choice(["slopes", "slopes", "none", "fast"])
    if kind == "linear":
        t = _log(rng, 1, 16384 if dtype == "f16" else 8192)
        return {"kind": kind, "dtype": dtype, "tokens": t, "requests": min(t, rng.choice([1, 1, rng.randint(2, 16)])),
                "uneven": rng.randint(6, 10 ** 6), "hk": hk, "hv": hv, "dk": dk, "dv": dv,
                "initial": rng.choice(["none", "shared", "own"]), "decay": decay}
    rows = _log(rng, 1, 128)
    padded = rng.choice([0, rng.randint(0, rows // 4)])
    case = {"kind": kind, "dtype": dtype, "rows": rows, "slots": rows + rng.choice([0, 0, rng.randint(1, 32)]),
            "padded": padded, "hk": hk, "hv": hv, "dk": dk, "dv": dv}
    return {**case, "decay": decay} if kind == "linear_step" else case


# --------------------------------------------------------------------------- sizes that follow from a case
def _offsets(case):
    """cu_seqlens of a linear case: uneven requests that add up to its tokens."""
    t, n = case["tokens"], case["requests"]
    cuts = sorted(random.Random(case["uneven"]).sample(range(1, t), n - 1)) if n > 1 else []
    return [0] + cuts + [t]


def _slots(case):
    """The pool slot of each row; -1 where a padded batch has no request."""
    rng = random.Random(case["rows"] * 1009 + case["slots"])
    rows = rng.sample(range(case["slots"]), case["rows"])
    empty = set(rng.sample(range(case["rows"]), case["padded"]))
    return [-1 if b in empty else slot for b, slot in enumerate(rows)]


def _shared(case):
    """(queries, own keys, first cache row) of each request; own keys count the queries' own."""
    rng = random.Random(case["uneven"])
    n, room = case["requests"], case["room"]
    queries = [min(room, rng.randint(1, case["tokens"])) for _ in range(n)]
    keys = [rng.randint(m, room) for m in queries]
    places = rng.sample(range(n), n)
    return queries, keys, [p * room for p in places]


# --------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def _decay(case, g):
    """Log-decays per head: a geometric range of memories (from about one token
    to a few hundred), no forgetting at all, or almost all of it."""
    h = torch.arange(1, case["hv"] + 1, device=DEV, dtype=torch.float32)
    jitter = 1.0 + 0.1 * torch.rand(case["hv"], generator=g, device=DEV)
    if case["decay"] == "none":
        return torch.zeros(case["hv"], device=DEV)
    if case["decay"] == "fast":
        return -3.0 * h * jitter
    return -torch.exp2(-8.0 * h / case["hv"]) * jitter


def prepare(case, seed):
    g = _gen(seed)
    kind, dt = case["kind"], DT[case["dtype"]]
    if kind == "shared":
        queries, keys, starts = _shared(case)
        n, t, room, p = len(queries), sum(queries), case["room"], case["prefix"]
        heads, kvh, d = case["heads"], case["kv_heads"], case["d"]
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
        cu = [sum(queries[:i]) for i in range(n + 1)]
        return {"case": case, "q": _randn(g, heads, t, d, dtype=dt), "gate": _randn(g, t, heads, d, dtype=dt),
                "prefix_k": _randn(g, kvh, p, d, dtype=dt),
                "prefix_vt": _randn(g, kvh, d, (p + 63) // 64 * 64, dtype=dt),
                "k": _randn(g, kvh, n * room, d, dtype=dt),
                "vt": _randn(g, kvh, d, (n * room + 63) // 64 * 64, dtype=dt),
                "cu": ints(cu), "start": ints(starts), "len": ints(keys)}
    hk, hv, dk, dv = (case[x] for x in ("hk", "hv", "dk", "dv"))
    t = case["tokens"] if kind == "linear" else case["rows"]
    s = {"case": case, "q": _randn(g, t, hk, dk, dtype=dt), "k": _randn(g, t, hk, dk, dtype=dt),
         "v": _randn(g, t, hv, dv, dtype=dt)}
    if kind == "linear":
        s["g"] = _decay(case, g)
        s["cu"] = torch.tensor(_offsets(case), dtype=torch.int32, device=DEV)
        shape = {"none": None, "shared": (hv, dk, dv), "own": (case["requests"], hv, dk, dv)}[case["initial"]]
        s["initial"] = None if shape is None else _randn(g, *shape)
        return s
    if kind == "linear_step":
        s["g"] = _decay(case, g)
    else:
        s["g"] = -torch.nn.functional.softplus(_randn(g, t, hv))
        s["beta"] = torch.sigmoid(_randn(g, t, hv))
    s["states"] = _randn(g, case["slots"], hv, dk, dv)
    # the pool that the new states go to, so that a draft can be taken back
    s["new"] = s["states"].clone()
    s["out"] = torch.zeros((t, hv, dv), dtype=dt, device=DEV)
    identity = case["slots"] == case["rows"] and not case["padded"]
    s["slots"] = None if identity else torch.tensor(_slots(case), dtype=torch.int32, device=DEV)
    return s


# --------------------------------------------------------------------------- one pass
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    clef = importlib.import_module("clef-rs_amd.clef_hip")
    case = s["case"]
    if case["kind"] == "shared":
        return clef.attention_gated_shared(s["q"], s["k"], s["vt"], s["gate"], s["cu"], s["start"], s["len"],
                                           prefix_k=s["prefix_k"], prefix_vt=s["prefix_vt"],
                                           max_keys=case["room"])
    if case["kind"] == "delta_step":
        out = clef.DeltaScan(case["dk"], case["dv"]).step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["states"],
                                                          slots=s["slots"], new_states=s["new"], out=s["out"])
        return {"out": out, "states": s["new"]}
    scan = clef.LinearScan(case["dk"], case["dv"])
    if case["kind"] == "linear_step":
        out = scan.step(s["q"], s["k"], s["v"], s["g"], s["states"], slots=s["slots"], new_states=s["new"],
                        out=s["out"])
        return {"out": out, "states": s["new"]}
    if case["requests"] == 1 and case["initial"] != "own":
        out, final = scan.prefill(s["q"], s["k"], s["v"], s["g"], initial=s["initial"], out_dtype=s["q"].dtype)
        return {"out": out, "final": final[None]}
    out, final = scan.prefill_varlen(s["q"], s["k"], s["v"], s["g"], s["cu"], initial=s["initial"],
                                     out_dtype=s["q"].dtype)
    return {"out": out, "final": final}


def _run_plain(s):
    kind = s["case"]["kind"]
    if kind == "shared":
        return _plain_shared(s)
    return _plain_linear(s) if kind == "linear" else _plain_step(s)


def _plain_linear(s):
    """Chunks of 128 packed tokens at once: products inside each chunk, one
    state per chunk, and the states of earlier chunks joined by a matrix of decays."""
    case, dt = s["case"], s["q"].dtype
    hv, n, t = case["hv"], case["requests"], case["tokens"]
    c = 128
    nc = -(-t // c)
    pad = nc * c - t
    rep = hv // case["hk"]
    g = s["g"].double()
    head = lambda x, r: torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, pad)).repeat_interleave(r, 1).transpose(0, 1)  # noqa: E731
    q, k, v = head(s["q"], rep) / math.sqrt(case["dk"]), head(s["k"], rep), head(s["v"], 1)  # [hv, nc * c, d]
    at = torch.arange(nc * c, device=DEV)
    cu = s["cu"].long()
    seq = torch.searchsorted(cu[1:], at, right=True)  # padding: a sequence of its own
    first, last = seq.view(nc, c)[:, 0], seq.view(nc, c)[:, -1]
    power = lambda e, keep: torch.where(keep, torch.exp(g.view(hv, *[1] * e.dim()) * e.clamp(min=0)), 0.0).float()  # noqa: E731
    # inside the chunks
    i = at[:c]
    sq = seq.view(nc, c)
    inner = power((i[:, None] - i[None, :])[None].expand(nc, c, c),
                  (i[:, None] >= i[None, :])[None] & (sq[:, :, None] == sq[:, None, :]))  # [hv, nc, c, c]
    qc, kc, vc = (x.reshape(hv, nc, c, -1) for x in (q, k, v))
    out = (qc @ kc.transpose(-1, -2) * inner) @ vc
    # what each chunk leaves, and what each chunk enters with
    left = (kc * power((c - 1 - i)[None].expand(nc, c), sq == last[:, None])[..., None]).transpose(-1, -2) @ vc
    cs = torch.arange(nc, device=DEV)
    joined = power((cs[:, None] - cs[None, :] - 1) * c, (cs[:, None] > cs[None, :]) & (first[:, None] == last[None, :]))
    enter = (joined @ left.reshape(hv, nc, -1)).view(hv, nc, case["dk"], case["dv"])
    out = out + (qc * power((i + 1)[None].expand(nc, c), sq == first[:, None])[..., None]) @ enter
    out = out.reshape(hv, nc * c, -1)[:, :t]
    # the initial states, and the final ones
    since = at[:t] - cu[seq[:t]] + 1
    until = cu[seq[:t] + 1] - 1 - at[:t]
    mine = seq[:t][None, :] == torch.arange(n, device=DEV)[:, None]
    weight = power(until[None].expand(n, t), mine).transpose(0, 1)  # [n, hv, t]
    final = (k[:, :t] * weight[..., None]).transpose(-1, -2) @ v[:, :t]
    if s["initial"] is not None:
        init = s["initial"].expand(n, hv, case["dk"], case["dv"])
        full = torch.ones_like(since, dtype=torch.bool)
        behind = q[:, :t] * power(since, full)[..., None]
        if case["initial"] == "shared":
            out = out + behind @ s["initial"]
        else:
            out = out + ((behind @ init) * mine[:, None, :, None]).sum(0)
        final = final + power(cu[1:] - cu[:-1], torch.ones_like(cu[1:], dtype=torch.bool)).t()[..., None, None] * init
    return {"out": out.transpose(0, 1).to(dt).contiguous(), "final": final}


def _plain_step(s):
    case = s["case"]
    hv, dk = case["hv"], case["dk"]
    rep = hv // case["hk"]
    q, k = (s[x].float().repeat_interleave(rep, 1) for x in "qk")
    v = s["v"].float()
    slots = torch.arange(case["rows"], device=DEV) if s["slots"] is None else s["slots"].long()
    state = s["states"][slots.clamp(min=0)]
    if case["kind"] == "delta_step":
        q = q / torch.sqrt(q.square().sum(-1, keepdim=True) + 1e-6) / math.sqrt(dk)
        k = k / torch.sqrt(k.square().sum(-1, keepdim=True) + 1e-6)
        state = state * torch.exp(s["g"])[..., None, None]
        d = (v - (state * k[..., None]).sum(-2)) * s["beta"][..., None]
        state = state + k[..., None] * d[..., None, :]
        out = (state * q[..., None]).sum(-2)
    else:
        state = state * torch.exp(s["g"])[:, None, None] + k[..., None] * v[..., None, :]
        out = (state * q[..., None]).sum(-2) / math.sqrt(dk)
    out = torch.where((slots >= 0)[:, None, None], out.to(s["out"].dtype), s["out"])
    if s["slots"] is None:
        return {"out": out, "states": state}
    named = slots[None, :] == torch.arange(case["slots"], device=DEV)[:, None]
    row = named.to(torch.uint8).argmax(1)
    return {"out": out, "states": torch.where(named.any(1)[:, None, None, None], state[row], s["new"])}


def _plain_shared(s):
    """Every query against the prefix and the whole cache, what is not its own masked."""
    case, dt = s["case"], s["q"].dtype
    rep, p, kn = case["heads"] // case["kv_heads"], case["prefix"], s["k"].shape[1]
    t = s["q"].shape[1]
    cu, start, length = s["cu"].long(), s["start"].long(), s["len"].long()
    at = torch.arange(t, device=DEV)
    seq = torch.searchsorted(cu[1:], at, right=True)
    end = start[seq] + length[seq] - (cu[seq + 1] - 1 - at)  # one behind the last key that a query sees
    key = torch.arange(kn, device=DEV)
    seen = (key[None, :] >= start[seq][:, None]) & (key[None, :] < end[:, None])
    seen = torch.cat([torch.ones((t, p), dtype=torch.bool, device=DEV), seen], 1)
    rows = s["q"].float().view(case["kv_heads"], rep, t, case["d"])
    keys = torch.cat([s["prefix_k"], s["k"]], 1).float()[:, None]
    values = torch.cat([s["prefix_vt"][:, :, :p], s["vt"][:, :, :kn]], 2).float()[:, None]
    scores = rows @ keys.transpose(-1, -2) / math.sqrt(case["d"])
    scores = torch.where(seen, scores, float("-inf"))
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = (e @ values.transpose(-1, -2)) / e.sum(-1, keepdim=True)
    out = out.view(case["heads"], t, case["d"]).transpose(0, 1)
    return (out / (1.0 + torch.exp(-s["gate"].float()))).to(dt).reshape(t, -1)


# --------------------------------------------------------------------------- least work
def work(case):
    kind, e = case["kind"], BYTES[case["dtype"]]
    if kind == "shared":
        queries, keys, _ = _shared(case)
        t, d, heads, kvh, p = sum(queries), case["d"], case["heads"], case["kv_heads"], case["prefix"]
        pairs = sum(n * p + n * m - n * (n - 1) // 2 for n, m in zip(queries, keys))
        return {"bytes": e * (3 * t * heads * d + 2 * kvh * d * (p + sum(keys))), "flops": 4 * heads * d * pairs}
    hk, hv, dk, dv = (case[x] for x in ("hk", "hv", "dk", "dv"))
    token = e * (2 * hk * dk + 2 * hv * dv)
    state = 4 * hv * dk * dv
    if kind == "linear":
        first = {"none": 0, "shared": 1, "own": case["requests"]}[case["initial"]]
        return {"bytes": case["tokens"] * token + (case["requests"] + first) * state,
                "flops": 4 * case["tokens"] * hv * dk * dv}
    live = case["rows"] - case["padded"]
    if kind == "linear_step":
        return {"bytes": live * (token + 2 * state), "flops": 4 * live * hv * dk * dv}
    return {"bytes": live * (token + 8 * hv + 2 * state), "flops": 6 * live * hv * dk * dv}


# --------------------------------------------------------------------------- 64-bit results
def exact(case, seed):
    def linear(s):
        """The recurrence, token by token."""
        rep = case["hv"] // case["hk"]
        q, k, v = s["q"].double() / math.sqrt(case["dk"]), s["k"].double(), s["v"].double()
        lam = torch.exp(s["g"].double())[:, None, None]
        out = torch.empty_like(v)
        finals = []
        offsets = _offsets(case)
        for r in range(case["requests"]):
            state = torch.zeros((case["hv"], case["dk"], case["dv"]), dtype=torch.float64, device=DEV)
            if s["initial"] is not None:
                state += s["initial"].double() if case["initial"] == "shared" else s["initial"][r].double()
            for t in range(offsets[r], offsets[r + 1]):
                state.mul_(lam).add_(k[t].repeat_interleave(rep, 0)[:, :, None] * v[t][:, None, :])
                torch.bmm(q[t].repeat_interleave(rep, 0)[:, None, :], state, out=out[t][:, None, :])
            finals.append(state)
        return {"out": out, "final": torch.stack(finals)}

    def step(s):
        rep = case["hv"] // case["hk"]
        out, new = s["out"].double(), s["new"].double()
        rows = list(range(case["rows"])) if s["slots"] is None else s["slots"].tolist()
        for b, slot in enumerate(rows):
            if slot < 0:
                continue
            q, k = (s[x][b].double().repeat_interleave(rep, 0) for x in "qk")
            v, state = s["v"][b].double(), s["states"][slot].double()
            if case["kind"] == "delta_step":
                q = q / (q.square().sum(1, keepdim=True) + 1e-6).sqrt()
                k = k / (k.square().sum(1, keepdim=True) + 1e-6).sqrt()
                state = state * torch.exp(s["g"][b].double())[:, None, None]
                write = (v - torch.bmm(k[:, None], state)[:, 0]) * s["beta"][b].double()[:, None]
            else:
                state = state * torch.exp(s["g"].double())[:, None, None]
                write = v
            state = state + torch.bmm(k[:, :, None], write[:, None])
            out[b] = torch.bmm(q[:, None], state)[:, 0] / math.sqrt(case["dk"])
            new[slot] = state
        return {"out": out, "states": new}

    def shared(s):
        queries, keys, starts = _shared(case)
        rep, p, d = case["heads"] // case["kv_heads"], case["prefix"], case["d"]
        out = []
        t = 0
        for n, m, first in zip(queries, keys, starts):
            for i in range(n):
                sees = m - n + i + 1
                k = torch.cat([s["prefix_k"], s["k"][:, first:first + sees]], 1).double()
                v = torch.cat([s["prefix_vt"][:, :, :p], s["vt"][:, :, first:first + sees]], 2).double()
                q = s["q"][:, t].double().view(case["kv_heads"], rep, d)
                w = torch.softmax(torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(d), -1)
                y = torch.bmm(w, v.transpose(1, 2).contiguous()).view(case["heads"], d)
                out.append((y * torch.sigmoid(s["gate"][t].double())).reshape(-1))
                t += 1
        return torch.stack(out)

    s = prepare(case, seed)
    return {"linear": linear, "shared": shared}.get(case["kind"], step)(s)
