"""Linear attention and the single-token steps where it is easy to go wrong:
widths narrower than a vector beside wide ones, infinities and NaN in states,
values and keys, factors far above and below the range of f16, launches at the
limits, and tokens that are views of different buffers.

References and bounds as in test_linear_gpu; where they are narrower here, the
text of the test says why.
"""
import numpy as np
import pytest
import torch

from test_linear_gpu import _cuda, _inputs, _randn, _slopes, check, reference

gpu = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.fixture(scope="module")
def clef():
    import clef_hip
    clef_hip.lib()
    return clef_hip


# ---------------------------------------------------------------------------- widths
@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("dk,dv", [(100, 5), (12, 4), (4, 13), (33, 3), (3, 33), (127, 1), (1, 127), (128, 2),
                                   (2, 128)])
def test_one_narrow_width(clef, dk, dv, dtype):
    """One width below a 16-byte vector, the other above it and mostly no multiple of one."""
    Hk, Hv, lens = 2, 4, [70, 1, 0, 130]
    T = sum(lens)
    q, k, v = _inputs(dk, T, Hk, Hv, dk, dv, dtype)
    g, init = _slopes(Hv), _randn(5, Hv, dk, dv)
    scan = clef.LinearScan(dk, dv)
    cq, ck, cv, cg, ci = _cuda(q, k, v, g, init)
    out, final = scan.prefill(cq, ck, cv, cg, initial=ci, out_dtype=dtype)
    check(out, final, q, k, v, g, scan.scale, init)
    cu = np.concatenate([[0], np.cumsum(lens)])
    out, final = scan.prefill_varlen(cq, ck, cv, cg, torch.tensor(cu, dtype=torch.int32, device="cuda"), initial=ci,
                                     out_dtype=dtype)
    for s, n in enumerate(lens):
        a = int(cu[s])
        if n:
            check(out[a:a + n], final[s], q[a:a + n], k[a:a + n], v[a:a + n], g, scan.scale, init)
        else:
            assert torch.equal(final[s].cpu(), init)


# ---------------------------------------------------------------------------- states
@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("T", [1, 70, 900])
def test_infinite_state_entry_stays_in_its_column(clef, T, value, dtype):
    """One infinite or NaN entry of the initial state: the other value columns come out as without it."""
    H, dk, dv, row, col = 3, 64, 48, 7, 5
    q, k, v = _inputs(T, T, H, H, dk, dv, dtype)
    g = torch.tensor([-0.05, 0.0, -0.3])
    init = _randn(6, H, dk, dv)
    scan = clef.LinearScan(dk, dv)
    cq, ck, cv, cg = _cuda(q, k, v, g)
    clean, cfinal = scan.prefill(cq, ck, cv, cg, initial=init.cuda())
    check(clean, cfinal, q, k, v, g, scan.scale, init)
    init[1, row, col] = value
    out, final = scan.prefill(cq, ck, cv, cg, initial=init.cuda())
    hit = torch.zeros((H, dv), dtype=torch.bool, device="cuda")
    hit[1, col] = True
    assert torch.equal(out[:, ~hit], clean[:, ~hit])
    assert not torch.isfinite(out[:, hit]).any()
    entry = torch.zeros_like(final, dtype=torch.bool)
    entry[1, row, col] = True
    assert torch.equal(final[~entry], cfinal[~entry])
    assert torch.equal(final[entry].cpu(), torch.tensor([value])) or value != value and final[entry].isnan().all()


@gpu
@pytest.mark.parametrize("T", [3, 70, 500])
def test_state_columns_of_different_size(clef, T):
    """Each column of an f16 scan's state to its own scale, 2^-30 to 2^30 side by side.  The copy of the state
    is rounded relative to a column's largest entry, which is scaled to 2^13 or more, so the part below the
    normal range of f16 is off by at most 2^-25 2^-13 of that entry; here against the column's sums of
    absolute values, and with decays of 0, so that the entries stay where they are."""
    H, dk, dv = 2, 64, 32
    q, k, v = _inputs(T, T, H, H, dk, dv, F16)
    k[:] = 0  # the state alone
    g = torch.zeros(H)
    sizes = torch.exp2(torch.tensor([(-30, 30, 0, -15)[c % 4] for c in range(dv)], dtype=F32))
    init = _randn(6, H, dk, dv) * sizes
    scan = clef.LinearScan(dk, dv)
    out, final = scan.prefill(*_cuda(q, k, v, g), initial=init.cuda())
    assert torch.equal(final.cpu(), init)
    want, _ = reference(q, k, v, g, scan.scale, init)
    size, _ = reference(q.abs(), k, v, g, scan.scale, init.abs())
    top = init.abs().double().amax(1) * q.double().abs().sum(2).max() * scan.scale  # [H, dv]
    bound = (2.0 ** -11 + (dk + T + 8) * 2.0 ** -24) * size + 2.0 ** -38 * top
    err = (out.double().cpu() - want).abs()
    assert (err <= bound).all(), f"{float((err / bound).max()):.3g} of the bound"


def recurrence(q, k, v, g, scale, initial=None):
    """Token by token in 64 bits: infinities as the operator's definition has them."""
    T, Hv = v.shape[0], v.shape[1]
    rep = Hv // q.shape[1]
    q, k = (x.double().repeat_interleave(rep, 1) for x in (q, k))
    v, lam = v.double(), torch.exp(g.double())[:, None, None]
    s = torch.zeros((Hv, q.shape[2], v.shape[2]), dtype=torch.float64) if initial is None else initial.double()
    out = torch.empty(v.shape, dtype=torch.float64)
    for t in range(T):
        s = s * lam + k[t][:, :, None] * v[t][:, None, :]
        out[t] = scale * (q[t][:, :, None] * s).sum(1)
    return out, s


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("which", ["value", "key"])
@pytest.mark.parametrize("T,dk,dv", [(1, 1, 1), (70, 64, 64), (150, 40, 24), (300, 128, 128), (900, 100, 13)])
def test_infinities_in_the_state(clef, T, dk, dv, which, dtype):
    """An infinite value (key) makes its column (row) of the state infinite, not NaN, and so it stays; all
    factors are positive, so that outputs are infinite too wherever the recurrence has them so."""
    Hk, Hv = 1, 2
    q, k, v = (x.abs() + 0.125 for x in _inputs(T, T, Hk, Hv, dk, dv, dtype))
    at = [t for t in (T // 3, T // 2) if t < T]
    if which == "value":
        for n, t in enumerate(at):
            v[t, n % Hv, (3 * n + 1) % dv] = float("inf") * (1 - 2 * n)
    else:
        for n, t in enumerate(at):
            k[t, 0, (3 * n + 1) % dk] = float("inf")
    g = torch.tensor([-0.01, -0.2])
    scan = clef.LinearScan(dk, dv)
    cq, ck, cv, cg = _cuda(q, k, v, g)
    eo, ef = recurrence(q, k, v, g, scan.scale)
    mo, mf = eo.abs(), ef.abs()
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    for out, final in (scan.prefill(cq, ck, cv, cg), [x if i == 0 else x[0] for i, x in enumerate(
            scan.prefill_varlen(cq, ck, cv, cg, cu))]):
        out, final = out.double().cpu(), final.double().cpu()
        for got, want, size, rel in ((out, eo, mo, 2.0 ** -11 if dtype == F16 else 0.0), (final, ef, mf, 2.0 ** -21)):
            odd = ~torch.isfinite(want)
            assert torch.equal(got[odd & ~want.isnan()], want[odd & ~want.isnan()])
            assert torch.isnan(got[want.isnan()]).all()
            bound = ((dk + T + 8) * 2.0 ** -24 + rel) * size
            assert ((got - want).abs()[~odd] <= bound[~odd]).all()


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
def test_infinite_states_under_strong_decay(clef, dtype):
    """Where e^{g n} of a chunk or a unit leaves the range of f32, an infinite entry is still infinite."""
    T, H, d = 700, 1, 64
    q, k, v = (x.abs() + 0.125 for x in _inputs(1, T, H, H, d, d, dtype))
    v[10, 0, 3] = float("inf")
    g = torch.tensor([-5.0])
    init = _randn(2, H, d, d)
    init[0, 9, 8] = float("-inf")
    _, final = clef.LinearScan(d, d).prefill(*_cuda(q, k, v, g), initial=init.cuda())
    _, want = recurrence(q, k, v, g, d ** -0.5, init)
    final = final.double().cpu()
    odd = ~torch.isfinite(want)
    assert odd.sum() == d + 1 and torch.equal(final[odd], want[odd])
    assert ((final - want).abs()[~odd] <= ((d + T + 8) * 2.0 ** -24 + 2.0 ** -21) * want.abs()[~odd]).all()


# ---------------------------------------------------------------------------- single tokens
@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("dk", [1, 40, 128])
def test_step_after_an_infinite_value(clef, dk, dtype):
    """Two tokens of one request in one call, an infinite value in the first: as one call for each."""
    H, dv, col = 2, 24, 3
    q, k, v = (x.abs() + 0.125 for x in _inputs(dk, 2, H, H, dk, dv, dtype))
    v[0, 1, col] = float("inf")
    g = _slopes(H).cuda()
    cq, ck, cv = _cuda(q, k, v)
    scan = clef.LinearScan(dk, dv)
    old = _randn(4, 1, H, dk, dv).abs().cuda()
    both, each = old.clone(), old.clone()
    out = scan.step(cq, ck, cv, g, both, slots=torch.zeros(2, dtype=torch.int32, device="cuda"))
    want = torch.cat([scan.step(cq[i:i + 1], ck[i:i + 1], cv[i:i + 1], g, each) for i in range(2)])
    assert torch.equal(both, each) and torch.equal(out, want)
    assert (out[:, 1, col] == float("inf")).all() and (both[0, 1, :, col] == float("inf")).all()
    rest = torch.ones((H, dv), dtype=torch.bool, device="cuda")
    rest[1, col] = False
    assert torch.isfinite(out[:, rest]).all()


# ---------------------------------------------------------------------------- ranges of f16
@gpu
@pytest.mark.parametrize("size", [2.0 ** -11, 2.0 ** -6, 1.0, 2.0 ** 8])
@pytest.mark.parametrize("T,d", [(33, 64), (64, 128), (300, 64)])
def test_scores_of_any_size(clef, T, d, size):
    """Queries and keys of about `size`: scores of f16 inputs from 2^-22 to beyond 65,504.  A score is rounded
    by 2^-11 of itself, or, below the normal range of f16, by 2^-25 where the largest score of its query in a
    block of keys is at least 2^-10, and elsewhere by 2^-25 2^-13 of that largest one: by 2^-15 of it at most."""
    Hk, Hv = 1, 2
    q, k, v = _inputs(T, T, Hk, Hv, d, d, F16)
    q, k = (q.float() * size).to(F16), (k.float() * size).to(F16)
    g = _slopes(Hv)
    scan = clef.LinearScan(d, d)
    out, final = scan.prefill(*_cuda(q, k, v, g))
    want, state = reference(q, k, v, g, scan.scale)
    mo, ms = reference(q.abs(), k.abs(), v.abs(), g, scan.scale)
    top = (q[:, 0].double().abs() @ k[:, 0].double().abs().t()).amax(1) * scan.scale  # [T]
    small = top[:, None, None] * v.double().abs().sum(0)[None]
    _, kept = reference(q.abs(), k.abs(), v.abs(), torch.zeros(Hv), scan.scale)  # no state of a chunk is larger
    enter = kept.amax() * q.double().abs().sum(2).max() * scan.scale
    bound = (2.0 ** -11 + (d + T + 8) * 2.0 ** -24) * mo + 2.0 ** -15 * small + 2.0 ** -38 * enter
    err = (out.double().cpu() - want).abs()
    assert (err <= bound).all(), f"{float((err / bound).max()):.3g} of the bound"
    sbound = ((d + T + 8) * 2.0 ** -24 + 2.0 ** -21) * ms + 2.0 ** -25 * k.double().abs().sum(0).max()
    assert ((final.double().cpu() - state).abs() <= sbound).all()


@gpu
def test_queries_of_different_size(clef):
    """A query of another size than its neighbours (2^-20 and 2^12 of them) changes its own row alone."""
    T, H, d = 130, 2, 64
    q, k, v = _inputs(3, T, H, H, d, d, F16)
    g = torch.tensor([-0.01, -0.5])
    scan = clef.LinearScan(d, d)
    clean, _ = scan.prefill(*_cuda(q, k, v, g))
    for at, factor in ((3, 2.0 ** -20), (70, 2.0 ** 12), (129, 2.0 ** -14)):
        other = q.clone()
        other[at] = (q[at].float() * factor).to(F16)
        out, _ = scan.prefill(*_cuda(other, k, v, g))
        rest = torch.arange(T, device="cuda") != at
        assert torch.equal(out[rest], clean[rest])
        eo, _ = reference(other, k, v, g, scan.scale)
        mo, _ = reference(other.abs(), k.abs(), v.abs(), g, scan.scale)
        err = (out.double().cpu() - eo).abs()[at]
        assert (err <= (2.0 ** -10 + (d + T + 8) * 2.0 ** -24) * mo[at]).all()


# ---------------------------------------------------------------------------- limits
@gpu
def test_most_sequences_of_most_heads(clef):
    """4,096 sequences of 256 heads at 128 x 128, the limits of a ragged batch, in units that are joined."""
    nseq, Hk, Hv, d, long = 4096, 1, 256, 128, 1300
    T = long + 64
    q, k, v = _inputs(3, T, Hk, Hv, d, d, F16)
    lens = [0] * nseq
    lens[7] = long
    for s in range(100, 164):
        lens[s] = 1
    cu = np.concatenate([[0], np.cumsum(lens)])
    g = _slopes(Hv)
    scan = clef.LinearScan(d, d)
    cq, ck, cv, cg = _cuda(q, k, v, g)
    out, none = scan.prefill_varlen(cq, ck, cv, cg, torch.tensor(cu, dtype=torch.int32, device="cuda"),
                                    want_final=False, out_dtype=F16)
    assert none is None
    check(out[:long, :2].contiguous(), None, q[:long], k[:long], v[:long, :2], g[:2], scan.scale)
    for t in (long, T - 1):
        check(out[t:t + 1], None, q[t:t + 1], k[t:t + 1], v[t:t + 1], g, scan.scale)


@gpu
def test_many_sequences_of_two_units(clef):
    """400 sequences of one head, each cut into two units, more than are joined side by side."""
    nseq, n, H, d = 400, 400, 1, 64
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn((nseq * n, H, d), generator=gen, device="cuda", dtype=F16) for _ in range(3))
    init = torch.randn((nseq, H, d, d), generator=gen, device="cuda")
    g = torch.tensor([-0.003])
    scan = clef.LinearScan(d, d)
    cu = torch.arange(0, nseq * n + 1, n, dtype=torch.int32, device="cuda")
    out, final = scan.prefill_varlen(q, k, v, g.cuda(), cu, initial=init)
    for s in (0, 143, 255, 256, 257, 399):
        part = slice(s * n, (s + 1) * n)
        check(out[part], final[s], q[part].cpu(), k[part].cpu(), v[part].cpu(), g, scan.scale, init[s].cpu())


# ---------------------------------------------------------------------------- views
@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
def test_one_token_from_different_buffers(clef, dtype):
    """A single row has no token stride: q, k, v (and g, beta) as rows of buffers of any pitch."""
    Hk, Hv, dk, dv = 2, 4, 64, 32
    q, k, v = _inputs(1, 1, Hk, Hv, dk, dv, dtype)
    g, gates, beta = _slopes(Hv), -_randn(2, 1, Hv).abs(), torch.sigmoid(_randn(3, 1, Hv))

    def view(x, pitch):  # the row as the second of a wider buffer
        n = x[0].numel()
        buf = torch.zeros((3, n + pitch), dtype=x.dtype, device="cuda")
        buf[1, :n] = x.reshape(-1).cuda()
        return torch.as_strided(buf, x.shape, (n + pitch,) + x.stride()[1:], n + pitch)

    cq, ck, cv = view(q, 8), view(k, 24), view(v, 40)
    state = _randn(4, 1, Hv, dk, dv).cuda()
    linear, delta = clef.LinearScan(dk, dv), clef.DeltaScan(dk, dv)
    packed = _cuda(q, k, v)
    a, b = state.clone(), state.clone()
    assert torch.equal(linear.step(cq, ck, cv, g.cuda(), a), linear.step(*packed, g.cuda(), b)) and torch.equal(a, b)
    a, b = state.clone(), state.clone()
    assert torch.equal(delta.step(cq, ck, cv, view(gates, 3), view(beta, 5), a),
                       delta.step(*packed, gates.cuda(), beta.cuda(), b)) and torch.equal(a, b)
    one, two = (linear.prefill(*x, g.cuda(), initial=state[0]) for x in ((cq, ck, cv), packed))
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    one, two = (linear.prefill_varlen(*x, g.cuda(), cu) for x in ((cq, ck, cv), packed))
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("scale", [1e-30, 1e-20, -3.0, 1e20])
def test_any_scale(clef, scale, dtype):
    """The scale of the outputs is any finite number: scores of 2^-100 and 2^66 keep f16's relative precision."""
    T, H, d = 150, 2, 64
    q, k, v = _inputs(4, T, H, H, d, d, dtype)
    init = _randn(6, H, d, d)
    g = torch.tensor([-0.01, -0.1])
    out, _ = clef.LinearScan(d, d, scale=scale).prefill(*_cuda(q, k, v, g), initial=init.cuda())
    want, _ = reference(q, k, v, g, scale, init)
    mo, _ = reference(q.abs(), k.abs(), v.abs(), g, abs(scale), init.abs())
    top = (q.double().abs().transpose(0, 1) @ k.double().abs().permute(1, 2, 0)).amax(2).t()[..., None] * abs(scale)
    rel = 2.0 ** -11 if dtype == F16 else 0.0
    bound = (rel + (d + T + 8) * 2.0 ** -24) * mo
    if dtype == F16:  # factors below f16's normal range, of the largest score and of the largest state entry
        kept = reference(q.abs(), k.abs(), v.abs(), torch.zeros(H), 1.0, init.abs())[1].amax()
        bound = bound + 2.0 ** -15 * top * v.double().abs().sum(0) + \
            2.0 ** -38 * kept * abs(scale) * q.double().abs().sum(2)[..., None]
    err = (out.double().cpu() - want).abs()
    assert (err <= bound).all(), f"{float((err / bound).max()):.3g} of the bound"


@gpu
@pytest.mark.parametrize("size", [1e28, 1e34])
def test_huge_states_beside_small_scores(clef, size):
    """The output of a state far beyond f16 next to scores that have to be scaled up."""
    T, H, d = 70, 1, 64
    q, k, v = _inputs(5, T, H, H, d, d, F16)
    q = (q.float() * 2.0 ** -6).to(F16)
    k = (k.float() * 2.0 ** -12).to(F16)
    init = _randn(6, H, d, d) * size
    init[:, :, ::2] = 0.0  # every other column has its scores alone
    g = torch.tensor([-0.05])
    scan = clef.LinearScan(d, d)
    out, _ = scan.prefill(*_cuda(q, k, v, g), initial=init.cuda())
    want, _ = reference(q, k, v, g, scan.scale, init)
    mo, _ = reference(q.abs(), k.abs(), v.abs(), g, scan.scale, init.abs())
    bound = (2.0 ** -10 + (d + T + 8) * 2.0 ** -24) * mo
    assert ((out.double().cpu() - want).abs() <= bound).all()
