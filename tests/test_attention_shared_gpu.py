"""Gated attention of a batch behind one shared prefix (clef_attention_gated_shared)
against softmax attention in 64 bits, request by request.

Bounds.  With M the softmax average of |v| and X = max |q|.|k| / sqrt(d) over the
keys, a score is off by at most (d + 4) 2^-24 X (f32 sums), which changes its weight
by as much of itself; the sums over n keys add n 2^-24; f16 factors (the weights
in the product with V) are off by at most 2^-11 of themselves or 2^-25 of the
largest.  The gate multiplies by at most 1.  An output of f16 adds 2^-11 of itself.
"""
import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.fixture(scope="module")
def clef():
    import clef_hip
    clef_hip.lib()
    return clef_hip


def _randn(gen, *shape, dtype=F32, std=1.0):
    return (torch.randn(shape, generator=gen) * std).to(dtype)


class Batch:
    """queries, lens, starts per request; a cache of `rows` rows whose unused ones hold NaN."""

    def __init__(self, dtype, heads, kvh, d, prefix, queries, lens, starts, rows, seed=0, std=1.0, behind=0):
        gen = torch.Generator().manual_seed(seed)
        self.dtype, self.heads, self.kvh, self.d, self.prefix = dtype, heads, kvh, d, prefix
        self.queries, self.lens, self.starts = queries, lens, starts
        self.T = sum(queries) + behind
        self.q = _randn(gen, heads, self.T, d, dtype=dtype, std=std)
        self.gate = _randn(gen, self.T, heads, 2 * d, dtype=dtype)
        self.pk = _randn(gen, kvh, prefix, d, dtype=dtype) if prefix else None
        self.pvt = torch.full((kvh, d, (prefix + 7) // 8 * 8), float("nan"), dtype=dtype) if prefix else None
        if prefix:
            self.pvt[:, :, :prefix] = _randn(gen, kvh, d, prefix, dtype=dtype)
        self.k = torch.full((kvh, rows, d), float("nan"), dtype=dtype)
        self.vt = torch.full((kvh, d, (rows + 7) // 8 * 8), float("nan"), dtype=dtype)
        for a, n in zip(starts, lens):
            self.k[:, a:a + n] = _randn(gen, kvh, n, d, dtype=dtype)
            self.vt[:, :, a:a + n] = _randn(gen, kvh, d, n, dtype=dtype)
        self.cu = np.concatenate([[0], np.cumsum(queries)])

    def cuda(self):
        ints = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
        dev = lambda x: None if x is None else x.cuda()  # noqa: E731
        return dict(q=dev(self.q), k=dev(self.k), vt=dev(self.vt), gate=self.gate.cuda()[:, :, self.d:],
                    cu_seqlens=ints(self.cu), key_starts=ints(self.starts), key_lens=ints(self.lens),
                    prefix_k=dev(self.pk), prefix_vt=dev(self.pvt))

    def reference(self, max_keys=None):
        """(y [rows, heads * d], its bound) in 64 bits."""
        rep, d = self.heads // self.kvh, self.d
        y, bound = [], []
        for s, (n, first) in enumerate(zip(self.queries, self.starts)):
            length = self.lens[s] if max_keys is None else min(self.lens[s], max_keys)
            for i in range(n):
                t, sees = int(self.cu[s]) + i, max(0, length - n + 1 + i)
                ks, vs = [self.k[:, first:first + sees]], [self.vt[:, :, first:first + sees]]
                if self.prefix:
                    ks, vs = [self.pk] + ks, [self.pvt[:, :, :self.prefix]] + vs
                k, v = torch.cat(ks, 1).double(), torch.cat(vs, 2).double().transpose(1, 2)
                gate = torch.sigmoid(self.gate[t, :, self.d:].double())
                if k.shape[1] == 0:
                    y.append(torch.zeros(self.heads * d, dtype=torch.float64))
                    bound.append(torch.zeros(self.heads * d, dtype=torch.float64))
                    continue
                q = self.q[:, t].double().view(self.kvh, rep, d)
                scores = q @ k.transpose(1, 2) / d ** 0.5
                w = torch.softmax(scores, -1)
                o = (w @ v).view(self.heads, d) * gate
                m = (w @ v.abs()).view(self.heads, d) * gate
                x = float((q.abs() @ k.abs().transpose(1, 2)).max()) / d ** 0.5
                rel = (2 * (d + 4) * x + 2 * k.shape[1] + 64) * 2.0 ** -24
                e = rel * m
                if self.dtype == F16:
                    small = (w.amax(-1, keepdim=True) * v.abs().sum(1)[:, None]).reshape(self.heads, d) * gate
                    e = e + 2.0 ** -11 * m + 2.0 ** -25 * small + 2.0 ** -11 * o.abs() + 2.0 ** -25
                y.append(o.reshape(-1))
                bound.append(e.reshape(-1))
        return torch.stack(y), torch.stack(bound)

    def check(self, y, max_keys=None):
        rows = sum(self.queries)
        want, bound = self.reference(max_keys)
        y = y[:rows].double().cpu()
        assert torch.isfinite(y).all()
        err = (y - want).abs()
        assert (err <= bound).all(), f"{float((err / bound.clamp(min=1e-300)).max()):.3g} of the bound"


def _batch(dtype, heads, kvh, d, prefix, queries, lens, gap=3, **kw):
    """Own keys in the cache in a mixed order, with gaps (so at odd places)."""
    n = len(queries)
    order = np.random.default_rng(n).permutation(n)
    starts, at = [0] * n, gap
    for s in order:
        starts[s] = at
        at += lens[s] + gap
    return Batch(dtype, heads, kvh, d, prefix, queries, lens, starts, at + gap, **kw)


CASES = [
    # heads, kvh, d, prefix, queries, lens
    (1, 1, 8, 1, [1], [1]),
    (16, 2, 256, 512, [1, 1], [1, 40]),
    (16, 2, 256, 777, [5, 1, 3, 1, 2, 1, 4], [5, 1, 150, 64, 33, 32, 31]),
    (8, 1, 128, 63, [1] * 9, [1, 2, 3, 31, 32, 33, 63, 64, 65]),
    (6, 2, 64, 65, [2, 1, 8], [2, 129, 20]),
    (4, 4, 72, 300, [1, 1, 1], [7, 1, 260]),
    (3, 1, 40, 1000, [16, 17], [16, 400]),
    (16, 2, 256, 2049, [1] * 33, [1 + 5 * i for i in range(33)]),
    (12, 1, 256, 130, [3] * 11, [3] * 11),
    (32, 1, 64, 700, [1, 2], [300, 2]),
    (2, 2, 248, 129, [70], [90]),
    (8, 1, 256, 1500, [1], [5]),
    (16, 2, 256, 513, [1, 1], [20, 3]),
    (2, 1, 128, 3001, [2, 1], [9, 40]),
    (4, 2, 64, 600, [1, 2, 1], [1500, 1100, 1]),
    (24, 1, 128, 530, [1, 1], [1200, 33]),
    (20, 1, 64, 40, [1, 3], [1, 100]),
]


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:4]) + f"-{len(c[4])}req")
def test_batch(clef, case, dtype):
    b = _batch(dtype, *case)
    args = b.cuda()
    y = clef.attention_gated_shared(**args, max_keys=max(b.lens))
    b.check(y)
    # a looser bound on the own keys changes how the work is split, not what it is
    b.check(clef.attention_gated_shared(**args))
    assert torch.equal(y, clef.attention_gated_shared(**args, max_keys=max(b.lens)))


SPLITS = [
    # heads, kvh, d, prefix, requests, tokens of each, own keys at most, rows behind the last sequence
    (4, 4, 64, 530, 60, 1, 200, 0),       # own keys beside the joining, 60 rows of a key head
    (8, 8, 72, 300, 9, 3, 90, 5),         # the same, a padded width, 32 rows
    (16, 2, 256, 600, 97, 1, 130, 70),
    (24, 24, 64, 257, 9, 1, 40, 0),       # 16 rows
    (12, 3, 128, 400, 5, 2, 70, 3),       # own keys as parts, 40 rows
    (5, 5, 128, 400, 13, 1, 1000, 2),     # 13 rows
    (34, 2, 64, 0, 40, 1, 300, 1),        # no prefix, 17 heads of a key head
    (34, 1, 40, 300, 3, 1, 300, 1),
]


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("split", SPLITS, ids=lambda c: "-".join(str(x) for x in c))
def test_split_of_the_own_keys(clef, split, dtype):
    heads, kvh, d, prefix, requests, tokens, most, behind = split
    lens = [max(tokens, 1 + (37 * s) % most) for s in range(requests)]
    b = _batch(dtype, heads, kvh, d, prefix, [tokens] * requests, lens, behind=behind)
    out = torch.full((b.T, heads * d), 7.0, dtype=dtype, device="cuda")
    y = clef.attention_gated_shared(**b.cuda(), max_keys=max(lens), out=out)
    b.check(y)
    assert (y[b.T - behind:] == 7.0).all()
    assert torch.equal(y, clef.attention_gated_shared(**b.cuda(), max_keys=max(lens), out=out.clone()))


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
def test_without_prefix_or_own_keys(clef, dtype):
    b = _batch(dtype, 8, 2, 128, 0, [1, 2, 1], [40, 130, 1])
    b.check(clef.attention_gated_shared(**b.cuda()))
    c = _batch(dtype, 8, 2, 128, 333, [1, 2, 1], [0, 0, 0])
    args = c.cuda()
    c.check(clef.attention_gated_shared(**args))
    c.check(clef.attention_gated_shared(**{**args, "k": None, "vt": None, "key_starts": None, "key_lens": None}))


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("prefix", [0, 100])
def test_queries_that_see_no_own_key(clef, prefix, dtype):
    """Fewer own keys than queries: the first queries see the prefix only, or nothing (zeros); empty requests."""
    b = _batch(dtype, 4, 2, 64, prefix, [4, 0, 3, 1], [2, 0, 0, 5], behind=2)
    out = torch.full((b.T, 4 * 64), 7.0, dtype=dtype, device="cuda")
    y = clef.attention_gated_shared(**b.cuda(), out=out)
    assert y is out and (y[-2:] == 7.0).all()
    b.check(y)
    if not prefix:
        assert (y[:2] == 0).all() and (y[4:7] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
def test_bounded_lengths(clef, dtype):
    """key_lens beyond max_keys are cut to it, and tables that do not fit stay inside the cache."""
    b = _batch(dtype, 4, 2, 64, 50, [1, 1, 1], [20, 90, 64])
    b.check(clef.attention_gated_shared(**b.cuda(), max_keys=64), max_keys=64)
    args = b.cuda()
    for starts, lens in (([-5, 10 ** 9, 2 ** 31 - 1], [10, 10, 10]), ([0, 170, 3], [-1, 2 ** 31 - 1, 10 ** 6])):
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        y = clef.attention_gated_shared(**{**args, "key_starts": ints(starts), "key_lens": ints(lens)})
        assert y.shape == (3, 256)
    y = clef.attention_gated_shared(**{**args, "cu_seqlens": torch.tensor([3, -7, 2 ** 31 - 1, 1], dtype=torch.int32,
                                                                          device="cuda")})
    torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
def test_masked_values_do_not_reach_a_query(clef, dtype):
    """A later token's infinities and NaN do not reach an earlier query of its request, nor another request."""
    b = _batch(dtype, 16, 2, 64, 40, [5, 1], [37, 9])
    clean, cb = b.cuda(), b
    want = clef.attention_gated_shared(**clean)
    cb.check(want)
    for value in (float("nan"), float("inf"), -65504.0 if dtype == F16 else torch.finfo(F32).min):
        args = b.cuda()
        last = b.starts[0] + 36
        args["k"][:, last] = value
        args["vt"][:, :, last] = value
        got = clef.attention_gated_shared(**args)
        assert torch.equal(got[:4], want[:4]) and torch.equal(got[5], want[5])


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
def test_peaked_and_flat_scores(clef, dtype):
    """Scores of hundreds (one key takes all) and scores of zero."""
    for std in (30.0, 0.0):
        b = _batch(dtype, 8, 2, 128, 500, [1, 2], [70, 200], std=std)
        b.check(clef.attention_gated_shared(**b.cuda()))


@gpu
def test_matches_the_prompt_form(clef):
    """Short requests whose own keys are their queries' own: attention_gated_varlen computes the same."""
    heads, kvh, d, prefix, lens = 16, 2, 256, 512, [1, 3, 2, 7, 1]
    b = _batch(F16, heads, kvh, d, prefix, lens, lens, gap=0)
    order = sorted(range(len(lens)), key=lambda s: b.starts[s])
    args = b.cuda()
    packed_k = torch.cat([args["k"][:, b.starts[s]:b.starts[s] + lens[s]] for s in range(len(lens))], 1).contiguous()
    packed_v = torch.zeros((kvh, d, 64), dtype=F16, device="cuda")
    packed_v[:, :, :sum(lens)] = torch.cat([args["vt"][:, :, b.starts[s]:b.starts[s] + lens[s]]
                                            for s in range(len(lens))], 2)
    assert len(order) == len(lens)
    want = clef.attention_gated_varlen(args["q"], packed_k, packed_v, args["gate"], args["cu_seqlens"],
                                       args["prefix_k"], args["prefix_vt"])
    got = clef.attention_gated_shared(**args)
    b.check(got)
    # the prompt form also rounds the attention and the gate to f16 before their product
    assert torch.allclose(got.float(), want.float(), rtol=2.0 ** -8, atol=2.0 ** -11)


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
def test_captured_graph_replays(clef, dtype):
    """A captured launch follows cu_seqlens, key_starts and key_lens as they change on the device."""
    shape = (dtype, 8, 2, 128, 300)
    first = Batch(*shape, [1, 1, 1, 1], [5, 9, 0, 64], [0, 64, 128, 192], 256)
    args = first.cuda()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        clef.attention_gated_shared(**args, max_keys=64)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    out = torch.zeros((4, 8 * 128), dtype=dtype, device="cuda")
    with torch.cuda.graph(graph):
        clef.attention_gated_shared(**args, max_keys=64, out=out)
    for i, (queries, lens, starts) in enumerate([([1, 1, 1, 1], [6, 10, 1, 64], [0, 64, 128, 192]),
                                                 ([2, 0, 1, 1], [40, 0, 33, 1], [3, 0, 100, 70]),
                                                 ([1, 1, 1, 1], [64, 64, 64, 64], [192, 128, 64, 0])]):
        b = Batch(*shape, queries, lens, starts, 256, seed=i + 1)
        for name, x in b.cuda().items():
            args[name].copy_(x)
        eager = clef.attention_gated_shared(**args, max_keys=64)
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), f"replay {i}"
        b.check(out)


@gpu
def test_two_streams_at_once(clef):
    a, b = (_batch(F16, 16, 2, 256, 600 + i, [1] * 5, [100] * 5, seed=i) for i in range(2))
    args = [a.cuda(), b.cuda()]
    want = [clef.attention_gated_shared(**x) for x in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(clef.attention_gated_shared(**args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


@gpu
@pytest.mark.parametrize("many", [True, False])
def test_offsets_past_32_bits(clef, many):
    """Prefix values of a key head over 2^32 bytes, and own keys behind 2^31 elements of the cache."""
    heads, d, prefix, own = (40 if many else 8), 64, 600, 70
    b = _batch(F16, heads, 1, d, prefix, [1], [own], gap=0)
    args = b.cuda()
    rows = (1 << 25) + 512
    free = torch.cuda.mem_get_info()[0]
    if free < 16 << 30:
        pytest.skip("needs 16 GiB of device memory")
    big_pvt = torch.empty((1, d, 1 << 25), dtype=F16, device="cuda")
    big_pvt[:, :, :prefix] = args["prefix_vt"][:, :, :prefix]
    k = torch.empty((1, rows, d), dtype=F16, device="cuda")
    vt = torch.empty((1, d, rows), dtype=F16, device="cuda")
    at = rows - own - 1
    k[:, at:at + own] = args["k"][:, b.starts[0]:b.starts[0] + own]
    vt[:, :, at:at + own] = args["vt"][:, :, b.starts[0]:b.starts[0] + own]
    vt[:, :, at + own:] = float("nan")
    y = clef.attention_gated_shared(args["q"], k, vt, args["gate"], args["cu_seqlens"],
                                    torch.tensor([at], dtype=torch.int32, device="cuda"), args["key_lens"],
                                    prefix_k=args["prefix_k"], prefix_vt=big_pvt, max_keys=128)
    b.check(y)
