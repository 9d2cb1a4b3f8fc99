"""The paged cache's calls at their edges: tables that do not fit beside pages of others,
lengths updated in place, requests that share pages."""
import pytest
import torch

import test_paged_gpu as base

gpu = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32
MIN, MAX = -2 ** 31, 2 ** 31 - 1
ints = base.ints


@pytest.fixture(scope="module")
def clef():
    import clef_hip
    clef_hip.lib()
    return clef_hip


def same(a, b):
    return torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0))


# Device tables that do not fit, of three requests with at most 15 pages of 16 keys and 22 tokens
BAD = [([0, 20, 3, 5], [5, 6, 240]), ([22, 22, 0, 0], [1, 2, MAX]), ([0, 9, 2, 4], [MAX, MAX, MAX]),
       ([0, 5, MIN, 22], [200, 240, 33]), ([MIN, MIN, MIN, MIN], [MAX, 0, 7]), ([0, MAX, MIN, MAX], [MIN, MAX, 241]),
       ([0, 22, 0, 22], [240, 240, 240]), ([-5, 3, 40, 2], [1, 500, MIN])]


@gpu
@pytest.mark.parametrize("dtype", [F16, F32], ids=str)
@pytest.mark.parametrize("rep", [1, 4])
@pytest.mark.parametrize("requests", [3, 70])
def test_bad_tables_beside_others(clef, dtype, rep, requests):
    """Page tables lie between rows that name pages of others: an index that left a request's table would
    find such a page.  Nothing of others changes, nor a row before or behind the batch's."""
    T, width, page, kvh, d, heads = 22, 15, 16, 2, 64, 2 * rep
    g = torch.Generator(device="cuda").manual_seed(rep)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    mine, others = requests * width, 40
    around = torch.randint(mine, mine + others, (requests + 20, width), generator=g, device="cuda").int()
    around[10:10 + requests] = torch.randperm(mine, generator=g, device="cuda").int().view(requests, width)
    table = around[10:10 + requests]
    to_around = torch.randint(mine, mine + others, (requests + 20, 3), generator=g, device="cuda").int()
    to_around[10:10 + requests] = torch.arange(requests * 3, device="cuda").int().view(requests, 3)
    total = mine + others
    w = torch.ones(d, device="cuda")
    for cu, lens in BAD:
        k, vt = randn(total, kvh, page, d), randn(total, kvh, d, page)
        to_k, to_vt = k.clone(), vt.clone()
        scores = torch.rand((total, kvh, page), generator=g, device="cuda")
        new, to_scores = torch.full_like(scores, 7.0), torch.full_like(scores, 7.0)
        before = [x.clone() for x in (k, vt, to_k, to_vt)]
        cu = ints((cu[:-1] + [22, 0, 9] * 30)[:requests] + cu[-1:])
        lens = ints((lens + [240, MAX, MIN] * 30)[:requests])
        cache, to = clef.PagedCache(k, vt), clef.PagedCache(to_k, to_vt)
        # each output between rows of its own
        q_all = torch.full((heads + 2, T, d), 7.0, dtype=dtype, device="cuda")
        y_all = torch.full((T + 40, heads * d), 7.0, dtype=dtype, device="cuda")
        lse_all = torch.full((T + 40, heads), 7.0, device="cuda")
        q = cache.append(randn(T, heads, d), randn(T, kvh, d), randn(T, kvh, d), w, w, cu, lens, table, 32, 1e4,
                         out=q_all[1:1 + heads])
        q.copy_(randn(heads, T, d))
        lse = lse_all[20:20 + T]
        for window, sinks in ((0, 0), (30, 4)):
            cache.attention_gated(q, randn(T, heads, d), cu, lens, table, window=window, sinks=sinks, lse=lse,
                                  out=y_all[20:20 + T])
            cache.add_weights(q, torch.zeros_like(lse), cu, lens, table, scores, new_scores=new, window=window, sinks=sinks)
        cache.evict(scores, lens, table, 40, to, to_around[10:10 + requests], to_scores, sinks=4, recent=8)
        torch.cuda.synchronize()
        for now, was in zip((k, vt, to_k, to_vt), before):
            assert same(now[mine:], was[mine:]), (cu.tolist()[:4], "a page of others")
        assert same(to_k[requests * 3:], before[2][requests * 3:]) and same(to_vt[requests * 3:], before[3][requests * 3:])
        assert (new[mine:] == 7.0).all() and (to_scores[requests * 3:] == 7.0).all()
        assert (q_all[0] == 7.0).all() and (q_all[-1] == 7.0).all()
        for x in (y_all, lse_all):
            assert (x[:20] == 7.0).all() and (x[20 + T:] == 7.0).all()


@gpu
@pytest.mark.parametrize("dtype", [F16, F32], ids=str)
def test_evict_lengths_in_place(clef, dtype):
    """Lengths updated where they stand: every key head still cuts from the old ones."""
    requests, budget, sinks, recent, kvh, page, d = 70, 48, 4, 8, 8, 16, 16
    lens = [budget // 2 + 13 * s for s in range(requests)]
    b = base.Batch([(0, m) for m in lens], page, kvh, d, dtype, seed=1)
    to = base.Batch([(0, min(m, budget)) for m in lens], page, kvh, d, dtype, seed=2)
    scores = torch.rand((b.total, kvh, page), generator=b.g, device="cuda")
    to_scores = torch.zeros((to.total, kvh, page), device="cuda")
    cache, target = clef.PagedCache(b.k, b.vt), clef.PagedCache(to.k, to.vt)
    want_lens, want = cache.evict(scores, b.len, b.table, budget, target, to.table, to_scores, sinks=sinks, recent=recent)
    pools = [x.clone() for x in (to.k, to.vt, to_scores)]
    for _ in range(5):
        length, keep = b.len.clone(), torch.empty_like(want)
        for x in (to.k, to.vt, to_scores):
            x.zero_()
        rc = clef.lib().clef_paged_evict(
            cache._at, b.table.data_ptr(), b.table.shape[1], length.data_ptr(), requests, scores.data_ptr(), budget, sinks,
            recent, target._at, to.table.data_ptr(), to.table.shape[1], to_scores.data_ptr(), length.data_ptr(),
            keep.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert rc == 0, clef.last_error()
        assert torch.equal(length, want_lens) and torch.equal(keep, want)
        for s, m in enumerate(lens):
            for x, y in zip((to.k, to.vt.transpose(2, 3), to_scores), (pools[0], pools[1].transpose(2, 3), pools[2])):
                assert same(to.read(x, s, min(m, budget)), to.read(y, s, min(m, budget)))


# (keys behind the shared ones, whose pages, how many pages of 32 keys, from which column)
SHARED = {
    "family": [(200, None, 0, 0), (130, 0, 3, 0), (70, None, 0, 0), (90, 2, 3, 0), (110, 2, 2, 1), (97, 0, 3, 0), (40, 3, 1, 0)],
    "all": [(96 + 7 * s, 0 if s else None, 3, 0) for s in range(9)],
    "hundred": [(65 + s % 40, s % 3 if s > 2 else None, 2, 0) for s in range(130)],
}


@gpu
@pytest.mark.parametrize("name", SHARED, ids=str)
@pytest.mark.parametrize("dtype,new,rep,d", [(F16, 1, 4, 64), (F16, 20, 8, 64), (F16, 33, 8, 256), (F32, 1, 3, 72),
                                             (F32, 20, 8, 128)], ids=str)
def test_weights_of_shared_pages(clef, name, dtype, new, rep, d):
    """Requests that share pages: each key's score is what the first request that has it gives with pages of
    its own, in place or not; the same in every run."""
    page, kvh = 32, 2
    shape = SHARED[name]
    new = min(new, 3) if len(shape) > 100 else new
    b = base.Batch([(min(new, 1 + 5 * s), m) for s, (m, *_) in enumerate(shape)], page, kvh, d, dtype, seed=d)
    heads = kvh * rep
    before = [torch.rand((kvh, m), generator=b.g, device="cuda") for m, *_ in shape]
    rows = [list(x) for x in b.rows]
    for s, (m, of, count, at) in enumerate(shape):
        if of is not None:
            rows[s][at:at + count] = rows[of][at:at + count]
        for j in range(m):  # a shared key is the same in all requests that have it
            first = next(i for i in range(s + 1) if shape[i][0] > j and rows[i][j // page] == rows[s][j // page])
            if first < s:
                for x in (b.keys, b.values, before):
                    x[s][:, j] = x[first][:, j]
    scores = torch.full((b.total, kvh, page), float("nan"), device="cuda")

    def fill():
        for s in range(len(shape)):
            b.fill(b.k, s, b.keys[s])
            b.fill(b.vt.transpose(2, 3), s, b.values[s])
            b.fill(scores, s, before[s])

    fill()
    cache = clef.PagedCache(b.k, b.vt)
    q, gate = b.randn(heads, b.T, d), b.randn(b.T, heads, d)
    lse = torch.zeros((b.T, heads), device="cuda")
    cache.attention_gated(q, gate, b.cu, b.len, b.table, lse=lse)
    own = cache.add_weights(q, lse, b.cu, b.len, b.table, scores, new_scores=torch.full_like(scores, 7.0))
    own = [b.read(own, s, m) for s, (m, *_) in enumerate(shape)]
    b.rows = rows
    for s, x in enumerate(rows):
        b.table[s, :len(x)] = ints(x)
    for x in (b.k, b.vt, scores):
        x.fill_(float("nan"))
    fill()
    want, held = torch.full_like(scores, 7.0), scores.clone()
    for s in reversed(range(len(shape))):  # the first request last: it stays
        b.fill(want, s, own[s])
        b.fill(held, s, own[s])
    for _ in range(4):
        got = cache.add_weights(q, lse, b.cu, b.len, b.table, scores, new_scores=torch.full_like(scores, 7.0))
        assert torch.equal(got, want)
        assert same(cache.add_weights(q, lse, b.cu, b.len, b.table, scores), held), "in place"
        for s in range(len(shape)):
            b.fill(scores, s, before[s])


@gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4)])
@pytest.mark.parametrize("dtype,page,kvh,rep,d", [(F16, 64, 2, 8, 64), (F16, 32, 1, 16, 128), (F16, 256, 3, 5, 24),
                                                  (F32, 64, 2, 8, 256), (F32, 16, 1, 10, 200), (F32, 128, 2, 3, 8)],
                         ids=str)
def test_weights_widths(clef, window, sinks, dtype, page, kvh, rep, d):
    """Accumulated weights in every instance: the bounds are those of test_paged_gpu.py."""
    base.test_weights(clef, window, sinks, dtype, page, kvh, rep, d)


def spread(b, gap):
    """b's pools as views of one buffer, with NaN between the pages: (keys, values)."""
    pool = torch.full((b.total, 2, b.k[0].numel() + gap), float("nan"), dtype=b.dtype, device="cuda")
    n = b.k[0].numel()
    pool[:, 0, :n], pool[:, 1, :n] = b.k.flatten(1), b.vt.flatten(1)
    return pool[:, 0, :n].unflatten(1, b.k.shape[1:]), pool[:, 1, :n].unflatten(1, b.vt.shape[1:])


@gpu
@pytest.mark.parametrize("dtype", [F16, F32], ids=str)
@pytest.mark.parametrize("requests", [[(1, 300), (2, 90)], [(40, 300), (20, 90), (0, 500)]], ids=str)
def test_weights_and_evict_of_spread_pools(clef, dtype, requests):
    b = base.Batch(requests, 16, 2, 64, dtype, seed=2)
    heads, budget = 8, 60
    q, gate, lse = b.randn(heads, b.T, 64), b.randn(b.T, heads, 64), torch.zeros((b.T, heads), device="cuda")
    scores = torch.rand((b.total, 2, 16), generator=b.g, device="cuda")
    to = base.Batch([(0, min(m, budget)) for _, m in requests], 16, 2, 64, dtype, seed=3)
    results = []
    for far in (False, True):
        cache = clef.PagedCache(*(spread(b, 24) if far else (b.k, b.vt)))
        target = clef.PagedCache(*(spread(to, 8) if far else (to.k.clone(), to.vt.clone())))
        cache.attention_gated(q, gate, b.cu, b.len, b.table, lse=lse)
        new = cache.add_weights(q, lse, b.cu, b.len, b.table, scores, new_scores=torch.zeros_like(scores))
        to_scores = torch.zeros((to.total, 2, 16), device="cuda")
        kept = cache.evict(new, b.len, b.table, budget, target, to.table, to_scores, sinks=4, recent=8)
        results.append((lse.clone(), new, to_scores, *kept, target.k.contiguous(), target.vt.contiguous()))
    for near, far in zip(*results):
        assert same(near, far)


@gpu
@pytest.mark.parametrize("dtype,d,kvh,bits", [(F16, 256, 4, 32), (F32, 256, 4, 32), (F16, 8, 4, 34)], ids=str)
def test_weights_and_evict_of_far_pages(clef, dtype, d, kvh, bits):
    """Pages whose keys, and at d = 8 scores (2^31 of them), lie behind what 32 bits count."""
    page, heads, budget = 64, 8, 100
    near = base.Batch([(1, 500), (20, 200)], page, kvh, d, dtype, seed=11)
    q, gate = near.randn(heads, near.T, d), near.randn(near.T, heads, d)
    scores = torch.rand((near.total, kvh, page), generator=near.g, device="cuda")
    to = ints([[0, 1], [2, 3]])
    more = (1 << bits) // (page * kvh * d) + 40
    results = []
    for shift in (4, more):  # the pages that evictions fill, then those of the requests
        k = torch.empty((shift + near.total, kvh, page, d), dtype=dtype, device="cuda")
        vt = torch.empty((shift + near.total, kvh, d, page), dtype=dtype, device="cuda")
        pool = torch.empty((shift + near.total, kvh, page), device="cuda")
        k[:4], vt[:4], pool[:4] = 9.0, 9.0, 9.0
        k[shift:], vt[shift:], pool[shift:] = near.k, near.vt, scores
        table = torch.where((near.table >= 0) & (near.table < near.total), near.table + shift, near.table)
        cache, lse = clef.PagedCache(k, vt), torch.zeros((near.T, heads), device="cuda")
        y = cache.attention_gated(q, gate, near.cu, near.len, table, lse=lse)
        cache.add_weights(q, lse, near.cu, near.len, table, pool)
        kept = cache.evict(pool, near.len, table, budget, cache, to, pool, sinks=4, recent=8)
        # and back, to far pages
        far = ints([[shift, shift + 1], [shift + 2, shift + 3]])
        again = cache.evict(pool, kept[0], to, 50, cache, far, pool, sinks=4, recent=8)
        torch.cuda.synchronize()
        results.append([x.clone() for x in (y, lse, *kept, *again, k[:4], vt[:4], pool[:4], k[shift:], vt[shift:], pool[shift:])])
        del k, vt, pool, cache
    for a, b in zip(*results):
        assert same(a, b)


@gpu
@pytest.mark.parametrize("dtype,d", [(F16, 64), (F16, 8), (F32, 16)], ids=str)
def test_most_rows(clef, dtype, d):
    """The most rows of a request that a call takes, 65,536 tokens of 256 heads on one key head, behind a window
    of 64: sampled tokens, and the weights of sampled keys, against 64 bits (bounds as in test_paged_gpu.py)."""
    T, heads, page, window = 65536, 256, 64, 64
    b = base.Batch([(T, T)], page, 1, d, dtype, seed=d)
    cache = clef.PagedCache(b.k, b.vt)
    q, gate = b.randn(heads, T, d), b.randn(T, heads, d)
    lse = torch.zeros((T, heads), device="cuda")
    y = cache.attention_gated(q, gate, b.cu, b.len, b.table, window=window, lse=lse).view(T, heads, d)
    new = cache.add_weights(q, lse, b.cu, b.len, b.table, torch.zeros((b.total, 1, page), device="cuda"), window=window)
    new = b.read(new, 0, T)[0]
    keys, values = b.keys[0][0].double(), b.values[0][0].double()

    def rows(t):  # scores [tokens, heads, window] of tokens t, and their bounds
        j = t[:, None] - torch.arange(window - 1, -1, -1, device="cuda")
        at = j.clamp(min=0)
        x = q[:, t].double().transpose(0, 1)
        z = torch.bmm(x, keys[at].transpose(1, 2).contiguous()) / d ** 0.5
        ds = (d + 2) * base.E * torch.bmm(x.abs(), keys[at].abs().transpose(1, 2).contiguous()) / d ** 0.5
        return j, at, torch.where((j >= 0)[:, None], z, -torch.inf), ds

    t = torch.tensor([0, 1, 62, 63, 64, 65, 4095, 32767, 32768, 40000, T - 65, T - 2, T - 1], device="cuda")
    j, at, z, ds = rows(t)
    ds = ds.amax(2)
    w = torch.softmax(z, 2)
    sig = torch.sigmoid(gate[t].double())
    want, most = torch.bmm(w, values[at]) * sig, torch.bmm(w, values[at].abs()) * sig
    rel = 2 * ds + 2.0 ** -14 + (window + 16) * base.E + (2.0 ** -11 if dtype == F16 else 0.0)
    base.close(y[t], want, most * rel[..., None] + base.HALF[dtype] * want.abs() + 2.0 ** -24 * (dtype == F16), "y")
    total = torch.logsumexp(z, 2)
    base.close(lse[t], total, ds + 2.0 ** -15 + (window + 16) * base.E + total.abs() * 2 * base.E, "lse")
    for key in (0, 1, 63, 64, 40000, T - 64, T - 1):
        t = torch.arange(key, min(key + window, T), device="cuda")
        j, _, z, ds = rows(t)
        z = z[j[:, None].expand_as(z) == key].view(len(t), heads)
        ds = ds[j[:, None].expand_as(ds) == key].view(len(t), heads)
        w = torch.exp(z - lse[t].double())
        want = w.sum()
        tol = (w * (2 * ds + 2.0 ** -14)).sum() + want * (heads * window + 8) * base.E
        base.close(new[key], want, tol, f"weight of key {key}")
