"""Attention behind a shared prefix at the limits of its launches and with tables
that do not fit the cache, against the same references as test_attention_shared_gpu.
"""
import pytest
import torch

from test_attention_shared_gpu import Batch

gpu = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.fixture(scope="module")
def clef():
    import clef_hip
    clef_hip.lib()
    return clef_hip


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
def test_one_token_of_strided_views(clef, dtype):
    """One query row: the gate may be a head-major view, whose token stride is shorter than a row, and out any row."""
    heads, kvh, d, prefix = 6, 2, 64, 40
    b = Batch(dtype, heads, kvh, d, prefix, [1], [9], [3], 16)
    args = b.cuda()
    want = clef.attention_gated_shared(**args)
    b.check(want)
    gate = args["gate"].transpose(0, 1).contiguous().transpose(0, 1)
    assert gate.stride() == (d, d, 1)
    out = torch.as_strided(torch.zeros(heads * d, dtype=dtype, device="cuda"), (1, heads * d), (1, 1))
    assert torch.equal(clef.attention_gated_shared(**{**args, "gate": gate}, out=out), want)


@gpu
@pytest.mark.parametrize("prefix,max_keys", [(16, 8), (0, 8), (300, 8), (300, 2000)],
                         ids=["short", "one launch", "beside", "parts"])
def test_most_tokens_of_most_heads(clef, prefix, max_keys):
    """65,536 tokens of 256 key heads, the limits of a call, in each of its forms.  An f16 output is off by 2^-11
    of itself, its f16 weights by 2^-11 of the sum of |v| under them or by 2^-25 of the largest, its f32 sums
    (and those of the f32 reference) by far less than another 2^-12."""
    T, heads, d, nseq, own = 65536, 256, 8, 16, 8
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB of device memory")
    gen = torch.Generator(device="cuda").manual_seed(prefix)
    randn = lambda *shape: torch.randn(shape, generator=gen, device="cuda", dtype=F16)  # noqa: E731
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    q, gate = randn(heads, T, d), randn(T, heads, d)
    pk, pvt = randn(heads, prefix, d), randn(heads, d, (prefix + 7) // 8 * 8)
    before = dict(prefix_k=pk, prefix_vt=pvt) if prefix else {}
    k, vt = randn(heads, nseq * own, d), randn(heads, d, nseq * own)
    each = T // nseq
    y = clef.attention_gated_shared(q, k, vt, gate, ints([each * s for s in range(nseq + 1)]),
                                    ints([own * s for s in range(nseq)]), ints([own] * nseq), max_keys=max_keys,
                                    **before)
    for s in range(nseq):  # the last `own` queries of a request see own keys, 1 to all of them
        a, b = each * s, each * (s + 1)
        keys = torch.cat([pk, k[:, own * s:own * (s + 1)]], 1).float()
        values = torch.cat([pvt[:, :, :prefix], vt[:, :, own * s:own * (s + 1)]], 2).float()
        values = values.transpose(1, 2).contiguous()
        scores = q[:, a:b].float() @ keys.transpose(1, 2).contiguous() / d ** 0.5
        sees = (torch.arange(a, b, device="cuda") - (b - own) + 1).clamp(min=0)
        scores.masked_fill_(torch.arange(prefix + own, device="cuda")[None] >= prefix + sees[:, None], float("-inf"))
        w = torch.softmax(scores, -1).nan_to_num(0.0)  # no key: zeros
        g = torch.sigmoid(gate[a:b].float()).transpose(0, 1)
        want, size = (w @ values) * g, (w @ values.abs()) * g
        small = w.amax(-1, keepdim=True) * values.abs().sum(1)[:, None] * g
        bound = (2.0 ** -11 + 2.0 ** -12) * size + 2.0 ** -25 * small + 2.0 ** -11 * want.abs() + 2.0 ** -25
        err = (y[a:b].view(each, heads, d).transpose(0, 1).float() - want).abs()
        assert (err <= bound).all(), f"request {s}: {float((err / bound).max()):.3g} of the bound"


TABLES = [
    # heads, kvh, d, prefix, requests, rows of the cache, max_keys
    (4, 2, 64, 50, 5, 176, 176),       # one launch
    (16, 2, 256, 600, 5, 176, 100),    # own keys as parts, 40 rows of a key head
    (16, 2, 256, 600, 97, 176, 130),   # beside the joining, 128-row groups
    (4, 4, 72, 300, 9, 176, 90),       # as parts, 16-row groups of a padded width
    (8, 8, 72, 300, 30, 2048, 1500),   # long own keys in many parts
]


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("table", TABLES, ids=lambda c: "-".join(str(x) for x in c))
def test_starts_and_lengths_that_do_not_fit(clef, table, dtype):
    """key_starts and key_lens outside the cache: cut to it, in every form of the call."""
    heads, kvh, d, prefix, requests, rows, max_keys = table
    b = Batch(dtype, heads, kvh, d, prefix, [1] * requests, [rows] + [0] * (requests - 1), [0] * requests, rows)
    odd = [(-5, 10), (10 ** 9, 10), (2 ** 31 - 1, 10), (-2 ** 31, 2 ** 31 - 1), (0, -1), (rows - 6, 2 ** 31 - 1),
           (3, 10 ** 6), (rows, 1), (rows - 1, 1), (17, -2 ** 31), (rows // 2, rows)]
    pairs = [odd[s % len(odd)] for s in range(requests)]
    args = b.cuda()
    args["key_starts"], args["key_lens"] = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in zip(*pairs))
    b.starts = [min(max(a, 0), rows) for a, _ in pairs]
    b.lens = [min(max(n, 0), max_keys, rows - a) for a, (_, n) in zip(b.starts, pairs)]
    b.check(clef.attention_gated_shared(**args, max_keys=max_keys))


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [64, 72])
def test_many_far_keys_beside_a_near_one(clef, d, dtype):
    """2^18 keys 17.5 below the score of one: each has a weight of 2^-25.2 of the largest, all of them 0.66 % of the
    sum.  Rows enough that no work-group has fewer than all keys.  A weight is rounded to f16 by 2^-11 of itself
    or by 2^-25 of 2^-7 of the row's reference (the largest key's, or up to 2^8 times less), 2^-32 n = 2^-14 in
    all; scores and sums of n equal terms in f32 by 2^-24 of the score and, running, of n: 2^-18 and 2^-7 at the
    very worst, of these 0.66 %."""
    T, heads, n = 2100, 16, 1 << 18
    if dtype == F32:
        n = 1 << 15
    gap = 17.5
    q = torch.zeros((heads, T, d), dtype=dtype, device="cuda")
    q[:, :, 0] = 16.0
    pk = torch.zeros((1, n, d), dtype=dtype, device="cuda")
    pk[0, 3, 0] = gap * d ** 0.5 / 16
    pvt = torch.ones((1, d, n), dtype=dtype, device="cuda")
    pvt[0, :, 3] = 0.0
    gate = torch.full((T, heads, d), 100.0, dtype=dtype, device="cuda")  # open
    cu = torch.arange(T + 1, dtype=torch.int32, device="cuda")
    y = clef.attention_gated_shared(q, None, None, gate, cu, None, None, prefix_k=pk, prefix_vt=pvt)
    far = (n - 1) * torch.exp(-q[0, 0, 0].double() * pk[0, 3, 0].double() / d ** 0.5)
    want = far / (1 + far)
    bound = want * (2.0 ** -10 + 2.0 ** -18 + 2.0 ** -7) + 2.0 ** -14
    assert ((y.double() - want).abs() <= bound).all(), f"{float(y.double().mean())} for {float(want)}"
