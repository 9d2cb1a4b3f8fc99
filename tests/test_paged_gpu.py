"""The paged cache's calls against their definitions in 64 bits: append (norm, rotary
axes, pages), attention (chunks, single tokens, windows and sinks), accumulated
weights, eviction.  Everything that no query of a request sees (slots behind its last
key, keys its window has left, pages of nobody, table entries behind the last) holds
NaN or names no page.

Bounds.  With e = 2^-24 (f32's half step), a score q.k / sqrt(d) is off by at most
ds = (d + 2) e sum |q k| / sqrt(d) (f32 sums of exact or once rounded products), and the
exponential's argument is formed in log2 units below 2^8 in size, off by 2^8 e = 2^-16
at most; a weight is off by the factor 1 + 2 ds + 2^-15.  f16 weights are rounded once
(2^-11; those below 2^-22 of the reference to a step of 2^-31: of at most 4,096 keys
2^-19 in all).  Sums of n terms add n e.  So with A the same output over |v|,
|y' - y| <= A (2^-11 [f16] + 2 ds + 2^-14 + (n + 16) e) + half a step of y."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
E = 2.0 ** -24
HALF = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
NAN = float("nan")


@pytest.fixture(scope="module")
def clef():
    import clef_hip
    clef_hip.lib()
    return clef_hip


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Batch:
    """Requests of (new tokens, keys) in a shuffled pool of pages."""

    def __init__(self, requests, page, kvh, d, dtype, seed=0, spare=2, tail=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g, self.requests, self.page, self.kvh, self.d, self.dtype = g, requests, page, kvh, d, dtype
        counts = [-(-m // page) for _, m in requests]
        width, total = max(max(counts), 1) + spare, sum(counts) + spare
        order = torch.randperm(total, generator=g, device="cuda").tolist()
        self.rows = []
        for c in counts:
            self.rows.append(order[:c])
            order = order[c:]
        junk = [-1, total, 2 ** 31 - 1, -2 ** 31]
        self.table = ints([r + [junk[(i + s) % 4] for i in range(width - len(r))] for s, r in enumerate(self.rows)])
        self.total = total
        # keys and values, and the pools with NaN all around them
        self.keys = [self.randn(kvh, m, d) for _, m in requests]
        self.values = [self.randn(kvh, m, d) for _, m in requests]
        self.k = torch.full((total, kvh, page, d), NAN, dtype=dtype, device="cuda")
        self.vt = torch.full((total, kvh, d, page), NAN, dtype=dtype, device="cuda")
        for s in range(len(requests)):
            self.fill(self.k, s, self.keys[s])
            self.fill(self.vt.transpose(2, 3), s, self.values[s])
        self.new = [n for n, _ in requests]
        self.T = sum(self.new) + tail
        self.cu = ints([sum(self.new[:i]) for i in range(len(requests) + 1)])
        self.len = ints([m for _, m in requests])

    def randn(self, *shape, std=1.0):
        return (torch.randn(shape, generator=self.g, device="cuda") * std).to(self.dtype)

    def fill(self, pool, s, rows):
        """rows [kvh, m, ..] to request s's slots of pool [pages, kvh, page, ..]."""
        for i, x in enumerate(self.rows[s]):
            part = rows[:, i * self.page:(i + 1) * self.page]
            pool[x, :, :part.shape[1]] = part

    def read(self, pool, s, m):
        if not m:
            return pool[:0].transpose(0, 1).reshape(self.kvh, 0, *pool.shape[3:])
        return torch.cat([pool[x] for x in self.rows[s][:-(-m // self.page)]], 1)[:, :m]

    def hide(self, window, sinks):
        """NaN in every slot that no query sees any more."""
        for s, (n, m) in enumerate(self.requests):
            seen = set()
            for i in range(n):
                p = m - n + i
                seen |= {j for j in range(p + 1) if not window or j > p - window or j < sinks}
            gone = [j for j in range(m) if j not in seen]
            if gone:
                keys, values = self.keys[s].clone(), self.values[s].clone()
                keys[:, gone] = NAN
                values[:, gone] = NAN
                self.fill(self.k, s, keys)
                self.fill(self.vt.transpose(2, 3), s, values)


def reference(b, q, gate, window, sinks):
    """(y, bound of its error, lse, bound, weights [per request], ds) in 64 bits; rows behind
    the last request are NaN."""
    heads, T, d = q.shape
    rep = heads // b.kvh
    y = torch.full((T, heads, d), NAN, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(y)
    lse = torch.full((T, heads), NAN, dtype=torch.float64, device="cuda")
    lse_bound = torch.zeros_like(lse)
    all_scores, b.ds = [], []
    t = 0
    for s, (n, m) in enumerate(b.requests):
        b.ds.append(0.0)
        p = torch.arange(m - n, m, device="cuda")[:, None]
        j = torch.arange(m, device="cuda")[None]
        seen = (j <= p) & ((j > p - window) | (j < sinks)) if window else j <= p
        scores = torch.full((heads, n, m), -math.inf, dtype=torch.float64, device="cuda")
        for h in range(heads):
            k, v = b.keys[s][h // rep].double(), b.values[s][h // rep].double()
            x = q[h, t:t + n].double()
            z = (x @ k.t()) / math.sqrt(d)
            ds = (d + 2) * E * (x.abs() @ k.t().abs()) / math.sqrt(d)
            ds = torch.where(seen, ds, 0.0).amax(1, keepdim=True) if m else torch.zeros((n, 1), device="cuda")
            b.ds[s] = max(b.ds[s], float(ds.max()) if n else 0.0)
            z = torch.where(seen, z, -math.inf)
            scores[h] = z
            l = torch.logsumexp(z, 1) if m else torch.full((n,), -math.inf, device="cuda")
            w = torch.where(seen & (l > -math.inf)[:, None], torch.exp(z - l[:, None]), 0.0)
            sig = torch.sigmoid(gate[t:t + n, h].double())
            y[t:t + n, h] = (w @ v) * sig
            most = (w @ v.abs()) * sig
            rel = 2 * ds + 2.0 ** -14 + (m + 16) * E + (2.0 ** -11 if q.dtype == torch.float16 else 0.0)
            bound[t:t + n, h] = most * rel + HALF[q.dtype] * y[t:t + n, h].abs() + 2.0 ** -24 * (q.dtype == torch.float16)
            lse[t:t + n, h] = l
            lse_bound[t:t + n, h] = ds[:, 0] + 2.0 ** -15 + (m + 16) * E + torch.where(l > -math.inf, l.abs(), 0.0) * 2 * E
        all_scores.append(scores)
        t += n
    return y, bound, lse, lse_bound, all_scores


def close(got, want, bound, what):
    same = (got.double() == want) | ((got.double() - want).abs() <= bound)
    assert same.all(), f"{what}: {int((~same).sum())} of {same.numel()} off, by " \
                       f"{float(((got.double() - want).abs() / bound.clamp(min=1e-30))[~same].max()):.3g} bounds"


def attend(clef, b, heads, window=0, sinks=0):
    q, gate = b.randn(heads, b.T, b.d), b.randn(b.T, heads, b.d)
    cache = clef.PagedCache(b.k, b.vt)
    out = torch.full((b.T, heads * b.d), 7.0, dtype=b.dtype, device="cuda")
    lse = torch.full((b.T, heads), 7.0, device="cuda")
    cache.attention_gated(q, gate, b.cu, b.len, b.table, window=window, sinks=sinks, lse=lse, out=out)
    torch.cuda.synchronize()
    y, bound, want, lse_bound, _ = reference(b, q, gate, window, sinks)
    t = sum(b.new)
    close(out.view(b.T, heads, b.d)[:t], y[:t], bound[:t], "y")
    close(lse[:t], want[:t], lse_bound[:t], "lse")
    assert (out[t:] == 7.0).all() and (lse[t:] == 7.0).all(), "rows behind the last request"
    return q, gate, lse, out


REQUESTS = {
    "one": [(1, 1)], "two keys": [(1, 2)], "700": [(1, 700)], "ends": [(1, 64), (1, 65), (1, 63), (1, 128), (1, 17)],
    "uneven": [(1, 3000), (1, 5), (1, 16), (1, 900)], "empty": [(0, 0), (1, 5), (0, 70), (3, 3), (0, 0)],
    "few": [(2, 90), (5, 5), (3, 200)], "chunk": [(33, 300)], "prompt": [(130, 130)], "behind": [(100, 1500)],
    "mixed": [(1, 1000), (130, 513), (1, 1), (0, 9), (40, 40), (1, 65)], "early": [(5, 2), (1, 0), (40, 3)],
}
F16, F32 = torch.float16, torch.float32


@gpu
@pytest.mark.parametrize("name", REQUESTS, ids=str)
@pytest.mark.parametrize("dtype,page,kvh,rep,d", [(F16, 64, 2, 8, 256), (F16, 16, 1, 4, 64), (F16, 32, 2, 3, 128),
                                                  (F32, 16, 2, 8, 256), (F32, 128, 1, 3, 64)], ids=str)
def test_attention(clef, name, dtype, page, kvh, rep, d):
    attend(clef, Batch(REQUESTS[name], page, kvh, d, dtype, seed=len(name), tail=3), kvh * rep)


@gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 4), (64, 0), (64, 70), (100, 1000), (16, 16), (2000, 4)])
@pytest.mark.parametrize("dtype,page,d", [(F16, 16, 64), (F16, 64, 256), (F32, 32, 64)], ids=str)
def test_window_and_sinks(clef, window, sinks, dtype, page, d):
    for requests in (REQUESTS["mixed"], REQUESTS["uneven"], [(300, 700)]):
        b = Batch(requests, page, 2, d, dtype, seed=window + sinks)
        b.hide(window, sinks)
        attend(clef, b, 8, window, sinks)


@gpu
@pytest.mark.parametrize("dtype", [F16, F32], ids=str)
@pytest.mark.parametrize("d", [8, 24, 40, 72, 104, 136, 200, 248])
def test_attention_widths(clef, dtype, d):
    attend(clef, Batch([(1, 200), (20, 70)], 16, 2, d, dtype, seed=d), 8)


@gpu
@pytest.mark.parametrize("dtype", [F16, F32], ids=str)
@pytest.mark.parametrize("kvh,rep", [(1, 1), (1, 24), (4, 4), (3, 17), (2, 128), (16, 1)])
def test_attention_heads(clef, dtype, kvh, rep):
    attend(clef, Batch([(1, 200), (9, 70), (1, 1)], 32, kvh, 64, dtype, seed=rep), kvh * rep)


@gpu
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_attention_pages(clef, page):
    for dtype in (F16, F32):
        attend(clef, Batch([(1, 700), (150, 400), (1, 256)], page, 2, 128, dtype, seed=page), 8)


@gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 4)])
@pytest.mark.parametrize("dtype,page,d", [(F16, 16, 64), (F16, 64, 256), (F16, 32, 72), (F32, 16, 128)], ids=str)
@pytest.mark.parametrize("requests", [[(5, 40)], [(100, 230), (3, 70), (60, 60)]], ids=str)
def test_infinite_and_nan_values(clef, window, sinks, dtype, page, d, requests):
    """Infinite and NaN values reach the rows that see their key, in their feature, and no
    others; everything else keeps the bits that it has with finite values there."""
    heads = 8
    b = Batch(requests, page, 2, d, dtype, seed=d)
    q, gate = b.randn(heads, b.T, d), b.randn(b.T, heads, d)
    cache = clef.PagedCache(b.k, b.vt)
    run = lambda: cache.attention_gated(q, gate, b.cu, b.len, b.table, window=window, sinks=sinks).view(b.T, heads, d)  # noqa: E731
    odd = [(0, 1, 3, math.inf), (0, 0, d - 1, -math.inf), (0, 1, 9, NAN), (0, 0, 0, math.inf), (0, 0, 0, NAN)]
    places = []
    for s, (n, m) in enumerate(requests):
        first = m - n
        for (_, kv, f, x), j in zip(odd, (first + n // 2, m - 1, first + 1, max(first - 1, 0), max(first - 2, 0))):
            places.append((s, kv, f, j, x))
            b.values[s][kv, j, f] = 0.0
        b.fill(b.vt.transpose(2, 3), s, b.values[s])
    plain = run()
    for s, kv, f, j, x in places:
        b.values[s][kv, j, f] = x
        b.fill(b.vt.transpose(2, 3), s, b.values[s])
    got = run()
    torch.cuda.synchronize()
    want = plain.float()
    t = 0
    for s, (n, m) in enumerate(requests):
        for s2, kv, f, j, x in places:
            if s2 != s:
                continue
            for i in range(n):
                p = m - n + i
                if j <= p and (not window or j > p - window or j < sinks):
                    # an infinity, or NaN where it meets NaN or the other infinity
                    want[t + i, kv * 4:kv * 4 + 4, f] += x
        t += n
    assert torch.equal(got.float().nan_to_num(5.0, 6.0, 7.0), want.nan_to_num(5.0, 6.0, 7.0))


@gpu
def test_many_requests(clef):
    """More requests than threads deal with at once, most of them short."""
    requests = [(s % 3, s % 3 + s * 7 % 90) for s in range(1500)]
    attend(clef, Batch(requests, 16, 1, 64, F16, seed=3), 2)


@gpu
@pytest.mark.parametrize("dtype", [F16, F32], ids=str)
def test_attention_views(clef, dtype):
    """Pools that skip between pages, a gate inside a projection, outputs inside wider rows."""
    b = Batch([(1, 300), (20, 90)], 16, 2, 64, dtype)
    pool = torch.full((b.total, 3, b.k[0].numel()), NAN, dtype=dtype, device="cuda")
    pool[:, 0], pool[:, 2] = b.k.flatten(1), b.vt.flatten(1)
    heads = 8
    q, packed = b.randn(heads, b.T, b.d), b.randn(b.T, heads, 2 * b.d + 8)
    plain = clef.PagedCache(b.k, b.vt).attention_gated(q, packed[:, :, 64:128].contiguous(), b.cu, b.len, b.table)
    views = clef.PagedCache(pool[:, 0].view(b.k.shape), pool[:, 2].view(b.vt.shape))
    wide = torch.full((b.T, heads * 64 + 24), 7.0, dtype=dtype, device="cuda")
    views.attention_gated(q, packed[:, :, 64:128], b.cu, b.len, b.table, out=wide[:, 8:8 + heads * 64])
    assert torch.equal(wide[:, 8:8 + heads * 64], plain)
    assert (wide[:, :8] == 7.0).all() and (wide[:, 8 + heads * 64:] == 7.0).all()


@gpu
@pytest.mark.parametrize("dtype", [F16, F32], ids=str)
def test_far_pages(clef, dtype):
    """Pages whose offsets pass 32 bits."""
    page, kvh, d = 64, 4, 256
    per = page * kvh * d
    total = (1 << 32) // per + 40
    b = Batch([(1, 500), (20, 200)], page, kvh, d, dtype, seed=11)
    k, vt = (torch.empty((total, *x.shape[1:]), dtype=dtype, device="cuda") for x in (b.k, b.vt))
    k[-b.total:], vt[-b.total:] = b.k, b.vt
    for x in (k, vt):
        x[:b.total] = 100.0  # where a 32-bit offset would land
    shift = total - b.total
    table = torch.where((b.table >= 0) & (b.table < b.total), b.table + shift, b.table)
    q, gate = b.randn(8, b.T, d), b.randn(b.T, 8, d)
    want = clef.PagedCache(b.k, b.vt).attention_gated(q, gate, b.cu, b.len, b.table)
    far = clef.PagedCache(k, vt)
    assert torch.equal(far.attention_gated(q, gate, b.cu, b.len, table), want)
    # and what enters there
    w = torch.ones(d, device="cuda")
    x, y, v = (b.randn(b.T, h, d) for h in (8, kvh, kvh))
    near = clef.PagedCache(b.k, b.vt)
    args = (x, y, v, w, w, b.cu, b.len)
    assert torch.equal(far.append(*args, table, 64, 1e7), near.append(*args, b.table, 64, 1e7))
    assert torch.equal(k[-b.total:].nan_to_num(5.0), b.k.nan_to_num(5.0))
    assert torch.equal(vt[-b.total:].nan_to_num(5.0), b.vt.nan_to_num(5.0))
    del k, vt, far


# --------------------------------------------------------------------------- append
def turned(x, w, pos, axis_of, rot, theta, eps):
    """(value, bound without its last rounding) of norm and rotary in 64 bits: the norm is off
    by at most (d / 2 + 8) e, sine and cosine by 2^-22 and the sum of two products by 2 e more."""
    x, d = x.double(), x.shape[-1]
    n = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    half = rot // 2
    i = torch.arange(half, device="cuda", dtype=torch.float64)
    angle = (pos.double()[axis_of].t() * theta ** (-2 * i / rot) if rot else pos.double()[:0].t().new_zeros(len(x), 0))
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = n[..., :half], n[..., half:2 * half]
    y = torch.cat([a * c - b * s, b * c + a * s, n[..., 2 * half:]], -1)
    size = torch.cat([a.abs() + b.abs()] * 2 + [n[..., 2 * half:].abs()], -1)
    return y, size * ((d / 2 + 16) * E + 2.0 ** -21)


@gpu
@pytest.mark.parametrize("axes,far", [(0, 0), (1, 0), (1, 10 ** 6), (3, 0), (4, 10 ** 7), (2, -500)])
@pytest.mark.parametrize("dtype,page,kvh,rep,d,rot", [(F16, 64, 2, 8, 256, 64), (F16, 16, 1, 3, 72, 72),
                                                      (F32, 32, 2, 2, 128, 32), (F32, 16, 4, 4, 64, 0),
                                                      (F16, 32, 1, 1, 8, 6)], ids=str)
def test_append(clef, axes, far, dtype, page, kvh, rep, d, rot):
    for requests in ([(1, 1)], [(1, 64), (1, 65)], REQUESTS["mixed"], REQUESTS["early"], [(300, 777)]):
        b = Batch(requests, page, kvh, d, dtype, seed=d + axes, tail=2)
        heads, theta, eps = kvh * rep, 1e7, 1e-6
        x = b.randn(b.T, 2 * heads * d + 2 * kvh * d + 3)  # an odd row: nothing is aligned
        q = x[:, :2 * heads * d].view(b.T, heads, 2 * d)[:, :, :d] if axes == 1 else b.randn(b.T, heads, d)
        k = x[:, 2 * heads * d:2 * heads * d + kvh * d].view(b.T, kvh, d)
        v = x[:, 2 * heads * d + kvh * d:-3].view(b.T, kvh, d)
        qw, kw = (1 + 0.1 * torch.randn(d, generator=b.g, device="cuda") for _ in range(2))
        index = torch.cat([torch.arange(m - n, m) for n, m in requests] + [torch.zeros(2)]).cuda().int()
        pos = index[None] if not axes else torch.randint(0, 4000, (axes, b.T), generator=b.g, device="cuda").int() + far
        axis_of = None if axes < 2 else [i % axes for i in range(rot // 2)]
        k0, v0 = b.k.clone(), b.vt.clone()
        out = torch.full((heads, b.T, d), 7.0, dtype=dtype, device="cuda")
        got = clef.PagedCache(b.k, b.vt).append(q, k, v, qw, kw, b.cu, b.len, b.table, rot, theta,
                                                positions=pos if axes else None, axis_of=axis_of, eps=eps, out=out)
        assert got is out
        torch.cuda.synchronize()
        axis = torch.tensor(axis_of or [0] * (rot // 2), dtype=torch.long, device="cuda")
        t = sum(b.new)
        y, bound = turned(q, qw, pos, axis, rot, theta, eps)
        close(out.transpose(0, 1)[:t], y[:t], (bound + HALF[dtype] * y.abs() + 2.0 ** -25)[:t], "q")
        assert (out[:, t:] == 7.0).all()
        y, bound = turned(k, kw, pos, axis, rot, theta, eps)
        bound = bound + HALF[dtype] * y.abs() + 2.0 ** -25
        t = 0
        for s, (n, m) in enumerate(requests):
            for i in range(n):
                j = m - n + i
                if j >= 0:
                    page_, slot = b.rows[s][j // page], j % page
                    close(b.k[page_, :, slot], y[t + i], bound[t + i], "k")
                    assert torch.equal(b.vt[page_, :, :, slot], v[t + i])
                    b.k[page_, :, slot], b.vt[page_, :, :, slot] = k0[page_, :, slot], v0[page_, :, :, slot]
            t += n
        assert torch.equal(b.k.nan_to_num(5.0), k0.nan_to_num(5.0)), "a slot of nobody's token was written"
        assert torch.equal(b.vt.nan_to_num(5.0), v0.nan_to_num(5.0)), "a slot of nobody's token was written"


@gpu
@pytest.mark.parametrize("tokens", [1, 3])
@pytest.mark.parametrize("requests", [64, 65, 200])
def test_append_many_requests(clef, tokens, requests):
    """Fewer and more requests than a wave has lanes, few tokens and many, empty ones among them."""
    shape = [((s + 1) % (tokens + 1), (s + 1) % (tokens + 1) + s * 5 % 37) for s in range(requests)]
    b = Batch(shape, 16, 2, 64, F16, seed=requests, tail=1)
    x, k, v = (b.randn(b.T, h, 64) for h in (4, 2, 2))
    w = torch.ones(64, device="cuda")
    out = torch.full((4, b.T, 64), 7.0, dtype=F16, device="cuda")
    clef.PagedCache(b.k, b.vt).append(x, k, v, w, w, b.cu, b.len, b.table, 32, 1e4, out=out)
    torch.cuda.synchronize()
    index = torch.cat([torch.arange(m - n, m) for n, m in shape] + [torch.zeros(1)]).cuda().int()[None]
    axis = torch.zeros(16, dtype=torch.long, device="cuda")
    t = sum(b.new)
    y, bound = turned(x, w, index, axis, 32, 1e4, 1e-6)
    close(out.transpose(0, 1)[:t], y[:t], (bound + HALF[F16] * y.abs() + 2.0 ** -25)[:t], "q")
    assert (out[:, t:] == 7.0).all()
    y, bound = turned(k, w, index, axis, 32, 1e4, 1e-6)
    bound = bound + HALF[F16] * y.abs() + 2.0 ** -25
    t = 0
    for s, (n, m) in enumerate(shape):
        if n:
            close(b.read(b.k, s, m)[:, m - n:].transpose(0, 1), y[t:t + n], bound[t:t + n], "k")
            assert torch.equal(b.read(b.vt.transpose(2, 3), s, m)[:, m - n:].transpose(0, 1), v[t:t + n])
            if m > n:
                assert torch.equal(b.read(b.k, s, m)[:, :m - n], b.keys[s][:, :m - n])
                assert torch.equal(b.read(b.vt.transpose(2, 3), s, m)[:, :m - n], b.values[s][:, :m - n])
        t += n


@gpu
@pytest.mark.parametrize("dtype", [F16, F32], ids=str)
@pytest.mark.parametrize("new", [1, 70])
def test_shared_pages(clef, dtype, new):
    """Requests whose tables begin with the same pages: each as it would be with its own."""
    shared, page = 96, 32
    b = Batch([(new, shared + new + 5 * s) for s in range(3)], page, 2, 64, dtype, seed=new)
    for s in (1, 2):
        b.keys[s][:, :shared], b.values[s][:, :shared] = b.keys[0][:, :shared], b.values[0][:, :shared]
        b.fill(b.k, s, b.keys[s])
        b.fill(b.vt.transpose(2, 3), s, b.values[s])
    q, gate = b.randn(8, b.T, 64), b.randn(b.T, 8, 64)
    cache = clef.PagedCache(b.k, b.vt)
    want = cache.attention_gated(q, gate, b.cu, b.len, b.table)
    table = b.table.clone()
    table[1:, :shared // page] = table[0, :shared // page]
    assert torch.equal(cache.attention_gated(q, gate, b.cu, b.len, table), want)


# --------------------------------------------------------------------------- weights
@gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4), (1, 0), (70, 200)])
@pytest.mark.parametrize("dtype,page,kvh,rep,d", [(F16, 64, 2, 8, 256), (F16, 16, 1, 3, 72), (F32, 32, 2, 4, 64),
                                                  (F32, 16, 1, 20, 128)], ids=str)
def test_weights(clef, window, sinks, dtype, page, kvh, rep, d):
    for name in ("one", "ends", "uneven", "empty", "mixed", "early", "behind"):
        b = Batch(REQUESTS[name], page, kvh, d, dtype, seed=window + d, tail=1)
        b.hide(window, sinks)
        heads = kvh * rep
        q, _, lse, _ = attend(clef, b, heads, window, sinks)
        scores = torch.full((b.total, kvh, page), NAN, device="cuda")
        before = [torch.rand((kvh, m), generator=b.g, device="cuda") for _, m in b.requests]
        for s, (n, m) in enumerate(b.requests):
            old = before[s].clone()
            old[:, max(m - n, 0):] = NAN  # what stands at the new tokens' keys does not count
            b.fill(scores, s, old)
        start = scores.clone()
        new = torch.full_like(scores, 7.0)
        cache = clef.PagedCache(b.k, b.vt)
        assert cache.add_weights(q, lse, b.cu, b.len, b.table, scores, new_scores=new, window=window, sinks=sinks) is new
        assert torch.equal(scores.nan_to_num(5.0), start.nan_to_num(5.0))
        cache.add_weights(q, lse, b.cu, b.len, b.table, scores, window=window, sinks=sinks)
        torch.cuda.synchronize()
        z = reference(b, q, torch.zeros((b.T, heads, d), device="cuda"), window, sinks)[4]
        t = 0
        for s, (n, m) in enumerate(b.requests):
            row = lse[t:t + n].double().t()[:, :, None]
            w = torch.where(z[s] > -math.inf, torch.exp(z[s] - row), 0.0)  # [heads, n, m]
            want = w.view(kvh, rep * n, m).sum(1)
            tol = want * (2 * b.ds[s] + 2.0 ** -14 + (rep * n + 8) * E)
            old = before[s].double()
            old[:, max(m - n, 0):] = 0.0
            want = want + old
            close(b.read(new, s, m), want, tol + 2 * E * want, "new scores")
            assert torch.equal(b.read(new, s, m), b.read(scores, s, m)), "in place"
            b.fill(new, s, torch.full((kvh, m), 7.0, device="cuda"))
            t += n
        assert (new == 7.0).all(), "a slot of nobody's key was written"


# --------------------------------------------------------------------------- eviction
def kept(scores, m, budget, sinks, recent):
    if m <= budget:
        return list(range(m))
    fixed = set(range(sinks)) | set(range(m - recent, m))
    key = lambda j: (scores[j] == scores[j], scores[j] if scores[j] == scores[j] else 0.0, -j)  # noqa: E731
    rest = sorted((j for j in range(m) if j not in fixed), key=key, reverse=True)
    return sorted(fixed | set(rest[:budget - len(fixed)]))


@gpu
@pytest.mark.parametrize("kind", ["random", "ties", "signs", "same"])
@pytest.mark.parametrize("dtype,page,kvh,d", [(F16, 64, 2, 256), (F16, 16, 1, 72), (F32, 32, 3, 40), (F16, 256, 2, 8)],
                         ids=str)
def test_evict(clef, kind, dtype, page, kvh, d):
    lens = [700, 1, 0, 64, 65, 2000, 17, 333, 17000 if d < 100 else 1025]
    for budget, sinks, recent in ((1, 0, 0), (64, 4, 16), (65, 65, 0), (300, 0, 300), (500, 100, 399), (17, 0, 1),
                                  (4000, 4, 40)):
        b = Batch([(0, m) for m in lens], page, kvh, d, dtype, seed=budget)
        scores = torch.full((b.total, kvh, page), NAN, device="cuda")
        mine = []
        for s, m in enumerate(lens):
            x = torch.randn((kvh, m), generator=b.g, device="cuda")
            if kind == "random":
                x = torch.exp(3 * x)
            elif kind == "ties":
                x = torch.round(x)
            elif kind == "same":
                x = torch.full_like(x, 0.25)
            else:
                odd = torch.tensor([0.0, -0.0, math.inf, -math.inf, NAN, 1e-42, -1e-42, 3e38], device="cuda")
                pick = torch.randint(0, 12, x.shape, generator=b.g, device="cuda")
                x = torch.where(pick < 8, odd[pick.clamp(max=7)], x)
            mine.append(x)
            b.fill(scores, s, x)
        counts = [min(m, budget) for m in lens]
        to = Batch([(0, c) for c in counts], page, kvh, d, dtype, seed=1, spare=-(-budget // page))
        to.k.fill_(7.0)
        to.vt.fill_(7.0)
        to_scores = torch.full((to.total, kvh, page), 7.0, device="cuda")
        new_lens, keep = clef.PagedCache(b.k, b.vt).evict(scores, b.len, b.table, budget, clef.PagedCache(to.k, to.vt),
                                                          to.table, to_scores, sinks=sinks, recent=recent)
        torch.cuda.synchronize()
        assert new_lens.tolist() == counts
        for s, m in enumerate(lens):
            k, v, x = to.read(to.k, s, counts[s]), to.read(to.vt.transpose(2, 3), s, counts[s]), to.read(to_scores, s, counts[s])
            for h in range(kvh):
                want = kept(mine[s][h].tolist(), m, budget, sinks, recent)
                assert keep[s, h].tolist() == want + [-1] * (budget - len(want)), (s, h)
                at = torch.tensor(want, dtype=torch.long, device="cuda")
                assert torch.equal(k[h], b.keys[s][h, at]) and torch.equal(v[h], b.values[s][h, at])
                assert torch.equal(x[h].nan_to_num(5.0), mine[s][h, at].nan_to_num(5.0))
            seven = torch.full((kvh, counts[s], d), 7.0, dtype=dtype, device="cuda")
            to.fill(to.k, s, seven)
            to.fill(to.vt.transpose(2, 3), s, seven)
            to.fill(to_scores, s, seven[:, :, 0].float())
        assert (to.k == 7.0).all() and (to.vt == 7.0).all() and (to_scores == 7.0).all()


# --------------------------------------------------------------------------- streams and captured launches
def step(clef, b, to, heads, x, state):
    """One step of a server: the tokens enter, attend, are weighed, and a cut copy is made."""
    cache = clef.PagedCache(b.k, b.vt)
    q = cache.append(x["q"], x["k"], x["v"], x["w"], x["w"], b.cu, b.len, b.table, 32, 1e7)
    y = cache.attention_gated(q, x["gate"], b.cu, b.len, b.table, window=90, sinks=4, lse=state["lse"])
    cache.add_weights(q, state["lse"], b.cu, b.len, b.table, state["scores"], new_scores=state["new"], window=90, sinks=4)
    lens, keep = cache.evict(state["new"], b.len, b.table, 48, clef.PagedCache(to.k, to.vt), to.table, state["to"],
                             sinks=4, recent=8)
    return {"q": q, "y": y, "lens": lens, "keep": keep, "k": b.k, "vt": b.vt, "new": state["new"], "to_k": to.k,
            "to_vt": to.vt, "to": state["to"]}


def setup(dtype, seed=5):
    heads, d, kvh, page = 8, 64, 2, 16
    b = Batch([(1, 200), (20, 70), (1, 33)], page, kvh, d, dtype, seed=seed)
    to = Batch([(0, 48)] * 3, page, kvh, d, dtype, seed=6)
    x = {n: b.randn(b.T, h, d) for n, h in (("q", heads), ("k", kvh), ("v", kvh), ("gate", heads))}
    x["w"] = torch.ones(d, device="cuda")
    state = {"lse": torch.zeros((b.T, heads), device="cuda"), "to": torch.zeros((to.total, kvh, page), device="cuda")}
    state["scores"] = torch.rand((b.total, kvh, page), generator=b.g, device="cuda")
    state["new"] = torch.zeros_like(state["scores"])
    return b, to, heads, x, state


@gpu
@pytest.mark.parametrize("dtype", [F16, F32], ids=str)
def test_captured_step(clef, dtype):
    """A captured step, replayed with other tokens, lengths and tables, equals the eager one."""
    b, to, heads, x, state = setup(dtype)
    step(clef, b, to, heads, x, state)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(clef, b, to, heads, x, state)
    for i in range(4):
        for n in ("q", "k", "v", "gate"):
            x[n].copy_(b.randn(*x[n].shape))
        b.len.copy_(ints([[200, 70, 33], [150, 20, 1], [1, 60, 20], [199, 71, 34]][i]))
        b.cu.copy_(ints([[0, 1, 21, 22], [0, 10, 20, 21], [0, 1, 2, 22], [0, 7, 7, 20]][i]))
        first = {n: t.clone() for n, t in captured.items()}
        k0, v0 = b.k.clone(), b.vt.clone()
        graph.replay()
        torch.cuda.synchronize()
        got = {n: t.clone() for n, t in captured.items()}
        for n in ("q", "y", "new", "to_k", "to_vt", "to"):
            captured[n].copy_(first[n])
        b.k.copy_(k0)
        b.vt.copy_(v0)
        eager = step(clef, b, to, heads, x, state)
        torch.cuda.synchronize()
        for n, t in eager.items():
            rows = slice(None)
            if n in ("q", "y"):  # rows behind the last request: as they were, so not the same in new tensors
                rows = slice(0, int(b.cu[-1]))
                a, c = (z.transpose(0, 1) if n == "q" else z for z in (got[n], t))
            else:
                a, c = got[n], t
            assert torch.equal(a[rows].nan_to_num(5.0), c[rows].nan_to_num(5.0)), (i, n)


@gpu
def test_two_streams(clef):
    """Two batches on two streams at once, each with its own workspace."""
    sets = [setup(F16, 5), setup(F32, 9)]
    want = []
    for s in sets:
        pools = [t.clone() for t in (s[0].k, s[0].vt)]
        out = step(clef, *s)
        torch.cuda.synchronize()
        want.append({n: t.clone() for n, t in out.items()})
        s[0].k.copy_(pools[0])
        s[0].vt.copy_(pools[1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(3):
        got = []
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(step(clef, *s))
    torch.cuda.synchronize()
    for a, c in zip(got, want):
        for n in c:
            assert torch.equal(a[n].nan_to_num(5.0), c[n].nan_to_num(5.0)), n


@gpu
@pytest.mark.parametrize("dtype", [F16, F32], ids=str)
def test_bad_tables_stay_inside(clef, dtype):
    """Tables that do not fit: other values, but the calls return and write no page of others."""
    b, to, heads, x, state = setup(dtype)
    for cu, lens in (([0, 5, 3, 22], [200, 70, 33]), ([-4, 9, 400, 2], [10 ** 9, -7, 33]), ([22, 22, 0, 0], [1, 2, 3]),
                     ([0, 2 ** 31 - 1, -2 ** 31, 22], [2 ** 31 - 1, -2 ** 31, 5])):
        b.cu.copy_(ints(cu))
        b.len.copy_(ints(lens))
        b.table.copy_(torch.randint(-2 ** 31, 2 ** 31 - 1, b.table.shape, generator=b.g, device="cuda").int())
        k0, v0 = b.k.clone(), b.vt.clone()
        step(clef, b, to, heads, x, state)
        torch.cuda.synchronize()
        assert torch.equal(b.k.nan_to_num(5.0), k0.nan_to_num(5.0)) and torch.equal(b.vt.nan_to_num(5.0), v0.nan_to_num(5.0))


# --- chunks in f32: tables wide enough for tiles of 64 rows
def widened(monkeypatch, page):
    import functools
    import sys
    monkeypatch.setattr(sys.modules[__name__], "Batch", functools.partial(Batch, spare=(1 << 16) // page))


@gpu
@pytest.mark.parametrize("name", ["chunk", "prompt", "behind", "mixed", "early"])
@pytest.mark.parametrize("page,kvh,rep,d", [(16, 2, 8, 256), (32, 1, 4, 64), (256, 2, 3, 128), (64, 3, 24, 40),
                                            (16, 2, 5, 72), (64, 1, 16, 200), (32, 4, 2, 8)])
def test_attention_wide_f32(clef, monkeypatch, name, page, kvh, rep, d):
    widened(monkeypatch, page)
    test_attention(clef, name, F32, page, kvh, rep, d)


@gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 4), (64, 70), (100, 1000), (2000, 4)])
@pytest.mark.parametrize("page,d", [(16, 256), (32, 64), (64, 104)])
def test_window_and_sinks_wide_f32(clef, monkeypatch, window, sinks, page, d):
    widened(monkeypatch, page)
    test_window_and_sinks(clef, window, sinks, F32, page, d)


@gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 4)])
@pytest.mark.parametrize("page,d", [(16, 128), (32, 72), (64, 256)])
def test_infinite_and_nan_values_wide_f32(clef, monkeypatch, window, sinks, page, d):
    widened(monkeypatch, page)
    test_infinite_and_nan_values(clef, window, sinks, F32, page, d, [(100, 230), (3, 70), (60, 60)])


@gpu
@pytest.mark.parametrize("requests", [[(300, 3000)], [(700, 700)], [(200, 1000), (90, 2500), (1, 4000)]], ids=str)
def test_long_chunks_f32(clef, requests):
    attend(clef, Batch(requests, 64, 2, 128, F32, seed=len(requests), spare=1000), 16)


@gpu
def test_captured_chunk_f32(clef):
    """A chunk in f32 in a captured launch whose lengths change between replays."""
    b = Batch([(80, 900), (64, 300)], 64, 2, 256, F32, seed=4, spare=1000)
    q, gate = b.randn(16, b.T, 256), b.randn(b.T, 16, 256)
    cache = clef.PagedCache(b.k, b.vt)
    lens = b.len.clone()
    out = torch.zeros((b.T, 16 * 256), device="cuda")
    run = lambda: cache.attention_gated(q, gate, b.cu, lens, b.table, out=out)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for less in (0, 100, 200, 0, 170):
        lens.copy_(b.len - less)
        out.fill_(9.0)
        graph.replay()
        got = out.clone()
        run()
        torch.cuda.synchronize()
        assert torch.equal(got, out)


@gpu
@pytest.mark.parametrize("dtype", [F16, F32], ids=str)
@pytest.mark.parametrize("requests", [[(1, 700), (3, 90)], [(120, 2000), (1, 30)]], ids=str)
def test_odd_addresses(clef, dtype, requests):
    """Gates and outputs that begin at any element, rows any distance apart."""
    heads, d = 8, 128
    b = Batch(requests, 64, 2, d, dtype, seed=3, spare=1000)
    q, wide = b.randn(heads, b.T, d), b.randn(b.T, heads * (d + 1) + 2)
    gate = wide[:, 1:1 + heads * (d + 1)].view(b.T, heads, d + 1)[:, :, :d]
    cache = clef.PagedCache(b.k, b.vt)
    want = cache.attention_gated(q, gate.contiguous(), b.cu, b.len, b.table)
    out = torch.full((b.T, heads * d + 7), 7.0, dtype=dtype, device="cuda")
    cache.attention_gated(q, gate, b.cu, b.len, b.table, out=out[:, 3:3 + heads * d])
    assert torch.equal(out[:, 3:3 + heads * d], want)
    assert (out[:, :3] == 7.0).all() and (out[:, 3 + heads * d:] == 7.0).all()
