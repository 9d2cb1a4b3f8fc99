"""The paged cache's calls together, as a server runs them: prompts enter in chunks and
attend, answers follow token by token, the weights that each step gives are added up,
caches are cut to a budget and the answers go on over what is left.

At every step the attention equals that of a flat 64-bit one over the keys that the
request still has, within the bounds of test_paged_gpu.py; scores are the sums of the
weights that the same flat attention gives; and what an eviction keeps is what those
scores say."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
HEADS, KVH, D, PAGE, ROT, THETA = 8, 2, 64, 16, 32, 1e7
REP = HEADS // KVH
E = 2.0 ** -24


@pytest.fixture(scope="module")
def clef():
    import clef_hip
    clef_hip.lib()
    return clef_hip


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Pool:
    """Pages of keys, values and scores, and who has which."""

    def __init__(self, clef, pages, dtype):
        self.k = torch.full((pages, KVH, PAGE, D), float("nan"), dtype=dtype, device="cuda")
        self.vt = torch.full((pages, KVH, D, PAGE), float("nan"), dtype=dtype, device="cuda")
        self.scores = torch.full((pages, KVH, PAGE), float("nan"), device="cuda")
        self.cache = clef.PagedCache(self.k, self.vt)
        self.free = list(range(pages))[::-1]

    def grow(self, rows, length):
        while len(rows) * PAGE < length:
            rows.append(self.free.pop())

    def rows(self, tables):
        width = max(len(t) for t in tables)
        return ints([t + [-1] * (width - len(t)) for t in tables])

    def read(self, pool, rows, m):
        return torch.cat([pool[x] for x in rows], 1)[:, :m]


@gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 4)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=str)
def test_prompts_answers_and_cuts(clef, dtype, window, sinks):
    g = torch.Generator(device="cuda").manual_seed(7)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    pool = Pool(clef, 64, dtype)
    tables = [[], [], []]
    lens, places = [0, 0, 0], [0, 0, 0]  # keys in the cache, and tokens so far (their positions)
    sums = [torch.zeros((KVH, 0), dtype=torch.float64, device="cuda") for _ in tables]
    norm = torch.ones(D, device="cuda")
    # chunks of prompts, single tokens, a request that waits
    steps = [[40, 7, 1], [33, 0, 90], [1, 1, 1], [1, 5, 0], "cut", [1, 1, 1], [2, 1, 30], "cut", [1, 1, 1]]
    for step in steps:
        if step == "cut":
            budget, recent = 32, 8
            fresh = [[], [], []]
            kept = [min(m, budget) for m in lens]
            for t, m in zip(fresh, kept):
                pool.grow(t, m)
            before = [[pool.read(x, t, m).clone() for x in (pool.k, pool.vt.transpose(2, 3), pool.scores)]
                      for t, m in zip(tables, lens)]
            new_lens, keep = pool.cache.evict(pool.scores, ints(lens), pool.rows(tables), budget, pool.cache,
                                              pool.rows(fresh), pool.scores, sinks=4, recent=recent)
            assert new_lens.tolist() == kept
            for s, (t, m) in enumerate(zip(fresh, lens)):
                score = before[s][2]
                for h in range(KVH):
                    fixed = set(range(min(4, m))) | set(range(max(0, m - recent), m))
                    rest = sorted((j for j in range(m) if j not in fixed), key=lambda j: (-float(score[h, j]), j))
                    want = list(range(m)) if m <= budget else sorted(fixed | set(rest[:budget - len(fixed)]))
                    assert keep[s, h].tolist() == want + [-1] * (budget - len(want))
                    at = torch.tensor(want, device="cuda")
                    for x, old in zip((pool.k, pool.vt.transpose(2, 3), pool.scores), before[s]):
                        assert torch.equal(pool.read(x, t, kept[s])[h], old[h, at])
                sums[s] = torch.stack([sums[s][h, keep[s, h, :kept[s]].long()] for h in range(KVH)])
                pool.free += tables[s]
            tables, lens = fresh, kept
            continue
        T = sum(step)
        lens = [m + n for m, n in zip(lens, step)]
        for t, m in zip(tables, lens):
            pool.grow(t, m)
        cu, key_lens, pages = ints([sum(step[:i]) for i in range(4)]), ints(lens), pool.rows(tables)
        positions = ints([places[s] + i for s, n in enumerate(step) for i in range(n)])
        places = [a + n for a, n in zip(places, step)]
        q = pool.cache.append(randn(T, HEADS, D), randn(T, KVH, D), randn(T, KVH, D), norm, norm, cu, key_lens, pages, ROT,
                              THETA, positions=positions)
        gate, lse = randn(T, HEADS, D), torch.zeros((T, HEADS), device="cuda")
        y = pool.cache.attention_gated(q, gate, cu, key_lens, pages, window=window, sinks=sinks, lse=lse)
        pool.cache.add_weights(q, lse, cu, key_lens, pages, pool.scores, window=window, sinks=sinks)
        torch.cuda.synchronize()
        t = 0
        for s, (n, m) in enumerate(zip(step, lens)):
            sums[s] = torch.cat([sums[s], torch.zeros((KVH, m - sums[s].shape[1]), dtype=torch.float64, device="cuda")], 1)
            if n == 0:
                continue
            keys, values = (pool.read(x, tables[s], m).double() for x in (pool.k, pool.vt.transpose(2, 3)))
            p = torch.arange(m - n, m, device="cuda")[:, None]
            j = torch.arange(m, device="cuda")[None]
            seen = (j <= p) & ((j > p - window) | (j < sinks)) if window else j <= p
            for h in range(HEADS):
                x, k, v = q[h, t:t + n].double(), keys[h // REP], values[h // REP]
                z = torch.where(seen, x @ k.t() / math.sqrt(D), -math.inf)
                ds = (D + 2) * E * float((x.abs() @ k.t().abs()).max()) / math.sqrt(D)
                w = torch.softmax(z, 1)
                sig = torch.sigmoid(gate[t:t + n, h].double())
                want, most = (w @ v) * sig, (w @ v.abs()) * sig
                half = 2.0 ** -11 if dtype == torch.float16 else E
                tol = most * (2 * ds + 2.0 ** -14 + (m + 16) * E + (half if half > E else 0.0)) + half * want.abs() + E
                got = y.view(T, HEADS, D)[t:t + n, h].double()
                assert ((got - want).abs() <= tol).all(), (step, s, h)
                sums[s][h // REP] += w.sum(0)
            t += n
            # a weight is off by its score's and its log-sum-exp's ds and by 2^-13 (exponential, sums of
            # up to 2^7 terms), where ds = 66 x 2^-24 sum |q k| / 8 < 2^-10 for sum |q k| < 2^11
            got = pool.read(pool.scores, tables[s], m).double()
            assert ((got - sums[s]).abs() <= sums[s] * (2.0 ** -9) + 2.0 ** -20).all(), (step, s)
