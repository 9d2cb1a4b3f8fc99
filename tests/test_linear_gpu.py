"""Linear attention with one decay per head (clef_linear_scan, its ragged form
and clef_linear_step) and the gated-DeltaNet step against the recurrences in 64
bits, computed here token by token or as the masked product they amount to.

Bounds.  Let M be the same sums over absolute values (of q, k, v and the
initial state), so that every product and partial sum of the operator is at
most M.  f32 inputs: an output is a sum of at most dk + T products of up to
four factors, so it is off by at most (dk + T + 8) 2^-24 M, and the states
likewise.  f16 inputs are exact factors; the score and the copy of the state
that become f16 factors are each off by at most 2^-11, one of them in each
product, and an f16 output by 2^-11 of itself; values below the normal range
of f16 are off by at most 2^-25 (scores, times the sum of |v|) and by 2^-25 of
the largest state entry (the scaled copy).  The f32 states of f16 inputs keep
the f32 bound, widened by 2^-21 M for factors held to 22 bits and, for factors
below 2^-3, whose lower half leaves f16's normal range, by 2^-25 of the sum of |v|.
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


def _randn(seed, *shape, dtype=F32, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def _slopes(hv):
    return -torch.exp2(-8.0 * torch.arange(1, hv + 1, dtype=F32) / hv)


def _inputs(seed, T, Hk, Hv, dk, dv, dtype):
    return (_randn(seed, T, Hk, dk, dtype=dtype), _randn(seed + 1, T, Hk, dk, dtype=dtype),
            _randn(seed + 2, T, Hv, dv, dtype=dtype))


def _power(g, n):
    """e^{g n} per head (rows) and count (columns); e^{-inf 0} = 1."""
    return torch.where(n == 0, 1.0, torch.exp(g.double()[:, None] * n.double().clamp(min=1)[None]))


def reference(q, k, v, g, scale, initial=None):
    """(out [T, Hv, dv], final [Hv, dk, dv]) in 64 bits as one masked product."""
    T, Hv = v.shape[0], v.shape[1]
    rep = Hv // q.shape[1]
    q, k, v = (x.double().transpose(0, 1) for x in (q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1), v))
    s0 = torch.zeros((Hv, q.shape[2], v.shape[2]), dtype=torch.float64) if initial is None else initial.double()
    i = torch.arange(T)
    decay = _power(g, i)  # [Hv, T]
    lag = (i[:, None] - i[None, :])
    mask = torch.where(lag >= 0, decay[:, lag.clamp(min=0)], 0.0)
    out = scale * ((q @ k.transpose(1, 2) * mask) @ v + (q @ s0) * _power(g, i + 1)[..., None])
    final = (k * decay.flip(1)[..., None]).transpose(1, 2) @ v + _power(g, torch.tensor([T]))[..., None] * s0
    return out.transpose(0, 1), final


def check(out, final, q, k, v, g, scale, initial=None):
    """Against the reference, within the bounds of the module's text."""
    T, dk = q.shape[0], q.shape[2]
    eo, ef = reference(q, k, v, g, scale, initial)
    mo, mf = reference(q.abs(), k.abs(), v.abs(), g, abs(scale), None if initial is None else initial.abs())
    sums = (dk + T + 8) * 2.0 ** -24
    bound, sbound = sums * mo, sums * mf
    if q.dtype == F16:
        largest = mf.max() if initial is None else torch.maximum(mf.max(), initial.abs().max().double())
        bound = bound + 2.0 ** -11 * mo + 2.0 ** -25 * (v.double().abs().sum(0)[None] +
                                                        q.double().abs().sum(2).max() * largest)
        sbound = sbound + 2.0 ** -21 * mf + 2.0 ** -25 * v.double().abs().sum(0)[:, None]
    if out.dtype == F16:
        bound = bound + 2.0 ** -11 * eo.abs() + 2.0 ** -25
    out = out.double().cpu()
    assert torch.isfinite(out).all()
    err = (out - eo).abs()
    assert (err <= bound).all(), f"out: {float((err / bound.clamp(min=1e-300)).max()):.3g} of the bound"
    if final is not None:
        err = (final.double().cpu() - ef).abs()
        assert (err <= sbound).all(), f"state: {float((err / sbound.clamp(min=1e-300)).max()):.3g} of the bound"


def _cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


# ---------------------------------------------------------------------------- prompts
SHAPES = [(1, 1, 1, 1, 1), (2, 1, 2, 8, 8), (33, 4, 4, 64, 64), (63, 2, 6, 40, 24), (64, 1, 1, 128, 128),
          (65, 1, 3, 100, 72), (127, 2, 2, 128, 13), (128, 1, 2, 64, 128), (129, 1, 1, 33, 31), (255, 1, 2, 128, 128),
          (256, 2, 4, 64, 64), (257, 1, 5, 128, 128), (511, 1, 1, 16, 128), (513, 2, 2, 128, 64), (1030, 1, 2, 128, 128)]


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("T,Hk,Hv,dk,dv", SHAPES)
def test_prompt(clef, T, Hk, Hv, dk, dv, dtype):
    q, k, v = _inputs(T, T, Hk, Hv, dk, dv, dtype)
    g = _slopes(Hv)
    init = _randn(5, Hv, dk, dv) if T % 2 else None
    scan = clef.LinearScan(dk, dv)
    cq, ck, cv, cg, ci = _cuda(q, k, v, g, init)
    out, final = scan.prefill(cq, ck, cv, cg, initial=ci, out_dtype=dtype)
    check(out, final, q, k, v, g, scan.scale, init)
    # without the final state, the same output; again, the same bits
    again, none = scan.prefill(cq, ck, cv, cg, initial=ci, out_dtype=dtype, want_final=False)
    assert none is None and torch.equal(again, out)


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("g", [0.0, -1e-4, -3.0, -1000.0, -3e38, float("-inf")])
@pytest.mark.parametrize("T", [1, 70, 700])
def test_decays(clef, T, g, dtype):
    """No forgetting, almost none, and all of it (also where g n leaves the range of f32)."""
    q, k, v = _inputs(T, T, 1, 2, 64, 64, dtype)
    gs = torch.tensor([g, -0.05])
    init = _randn(6, 2, 64, 64)
    scan = clef.LinearScan(64, 64, scale=0.5)
    out, final = scan.prefill(*_cuda(q, k, v, gs, init), out_dtype=F32)
    check(out, final, q, k, v, gs, 0.5, init)


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
def test_large_states(clef, dtype):
    """States far above and far below the range of f16."""
    T, H, d = 200, 3, 64
    q, k, v = _inputs(9, T, H, H, d, d, dtype)
    init = _randn(10, H, d, d) * torch.tensor([1e7, 1e-7, 0.0])[:, None, None]
    v[:, 1] *= 2.0 ** -10
    g = torch.tensor([-0.01, -0.001, 0.0])
    out, final = clef.LinearScan(d, d).prefill(*_cuda(q, k, v, g, init))
    scale = d ** -0.5
    for h in range(3):  # head by head, so that the bounds go by each head's own size
        check(out[:, h:h + 1], final[h:h + 1], q[:, h:h + 1], k[:, h:h + 1], v[:, h:h + 1], g[h:h + 1], scale,
              init[h:h + 1])


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("initial", ["none", "shared", "own"])
@pytest.mark.parametrize("lens", [[1], [1, 1, 1], [0, 5, 0, 0, 70, 1, 0], [300, 2, 256, 64, 0, 513], [257, 255, 1, 64]])
def test_ragged(clef, lens, initial, dtype):
    """Empty sequences, single tokens, and rows behind the last sequence (NaN, not to be read; out left as it was)."""
    Hk, Hv, dk, dv, behind = 2, 4, 64, 48, 3
    cu = np.concatenate([[0], np.cumsum(lens)])
    total, n = int(cu[-1]), len(lens)
    T = total + behind
    q, k, v = _inputs(n, T, Hk, Hv, dk, dv, dtype)
    for x in (q, k, v):
        x[total:] = float("nan")
    g = _slopes(Hv)
    init = {"none": None, "shared": _randn(3, Hv, dk, dv), "own": _randn(3, n, Hv, dk, dv)}[initial]
    out = torch.full((T, Hv, dv), 7.0, dtype=dtype, device="cuda")
    scan = clef.LinearScan(dk, dv)
    cq, ck, cv, cg, ci = _cuda(q, k, v, g, init)
    got, final = scan.prefill_varlen(cq, ck, cv, cg, torch.tensor(cu, dtype=torch.int32, device="cuda"), initial=ci,
                                     out=out)
    assert got is out and (out[total:] == 7.0).all()
    for s in range(n):
        a, b = int(cu[s]), int(cu[s + 1])
        i = init if init is None or initial == "shared" else init[s]
        if a == b:
            assert torch.equal(final[s].cpu(), torch.zeros((Hv, dk, dv)) if i is None else i)
        else:
            check(out[a:b], final[s], q[a:b], k[a:b], v[a:b], g, scan.scale, i)


@gpu
def test_infinities_stay_with_their_sequence(clef):
    """What one sequence holds does not reach its neighbours."""
    lens, H, d = [70, 130, 64, 40], 2, 64
    cu = np.concatenate([[0], np.cumsum(lens)])
    q, k, v = _inputs(1, int(cu[-1]), H, H, d, d, F16)
    v[int(cu[1]) + 90] = float("inf")
    k[int(cu[2]):int(cu[3])] = float("nan")
    g = _slopes(H)
    out, final = clef.LinearScan(d, d).prefill_varlen(*_cuda(q, k, v, g),
                                                      torch.tensor(cu, dtype=torch.int32, device="cuda"))
    for s in (0, 3):
        a, b = int(cu[s]), int(cu[s + 1])
        check(out[a:b], final[s], q[a:b], k[a:b], v[a:b], g, d ** -0.5)
    assert not torch.isfinite(final[1]).all() and not torch.isfinite(final[2]).all()


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_a_token_reaches_only_later_ones(clef, value, dtype):
    """An infinite or NaN value (key, query) changes nothing before its token, and is seen from it on."""
    T, H, d, at = 150, 2, 64, 77
    q, k, v = _inputs(2, T, H, H, d, d, dtype)
    g = _slopes(H)
    scan = clef.LinearScan(d, d)
    clean, _ = scan.prefill(*_cuda(q, k, v, g))
    for which in range(3):
        x = [y.clone() for y in (q, k, v)]
        x[which][at, 1, 5] = value
        out, _ = scan.prefill(*_cuda(*x, g))
        assert torch.equal(out[:, 0], clean[:, 0]) and torch.equal(out[:at, 1], clean[:at, 1])
        if which == 0:  # a query: its own row only
            assert torch.equal(out[at + 1:, 1], clean[at + 1:, 1]) and not torch.isfinite(out[at, 1]).any()
        elif which == 1:
            assert not torch.isfinite(out[at:, 1]).any()
        else:  # a value: its own column only
            rest = torch.arange(d, device="cuda") != 5
            assert torch.equal(out[:, 1, rest], clean[:, 1, rest]) and not torch.isfinite(out[at:, 1, 5]).any()


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
def test_views_and_alignment(clef, dtype):
    """q, k and v as views of one packed projection row, at odd strides and bases, out as a view too."""
    T, Hk, Hv, dk, dv = 150, 2, 4, 64, 64
    for base, extra in ((0, 0), (0, 3), (1, 0), (8, 8), (3, 5)):
        width = 2 * Hk * dk + Hv * dv + extra
        flat = _randn(base, base + T * width, dtype=dtype)
        cflat = torch.empty(flat.numel(), dtype=dtype, device="cuda").copy_(flat)
        cut = lambda f: [f[base:].view(T, width)[:, a:b].view(T, h, -1) for a, b, h in (  # noqa: E731
            (0, Hk * dk, Hk), (Hk * dk, 2 * Hk * dk, Hk), (2 * Hk * dk, width - extra, Hv))]
        q, k, v = cut(flat)
        rows = torch.zeros((T, Hv * dv + 1), dtype=dtype, device="cuda")
        out = rows[:, 1:].view(T, Hv, dv)
        g = _slopes(Hv)
        _, final = clef.LinearScan(dk, dv).prefill(*cut(cflat), g.cuda(), out=out)
        check(out, final, q, k, v, g, dk ** -0.5)
        assert (rows[:, 0] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
def test_resumed_prompt(clef, dtype):
    """A prompt in pieces, each from the state the last one left."""
    T, Hk, Hv, d = 600, 1, 2, 128
    q, k, v = _inputs(4, T, Hk, Hv, d, d, dtype)
    g = _slopes(Hv)
    scan = clef.LinearScan(d, d)
    cq, ck, cv, cg = _cuda(q, k, v, g)
    state, outs = None, []
    for a, b in ((0, 1), (1, 257), (257, 300), (300, 600)):
        o, state = scan.prefill(cq[a:b], ck[a:b], cv[a:b], cg, initial=state)
        outs.append(o)
    check(torch.cat(outs), state, q, k, v, g, scan.scale)


@gpu
def test_long_prompt_tail(clef):
    """2^17 tokens: the last ones see the remembered ones only, so a window of them is the reference."""
    T, H, d, w = 1 << 17, 2, 64, 600
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn((T, H, d), generator=gen, device="cuda", dtype=F16) for _ in range(3))
    g = torch.tensor([-0.2, -1.0])  # e^{-0.2 600} is far below 2^-25
    out, final = clef.LinearScan(d, d).prefill(q, k, v, g.cuda())
    eo, ef = reference(*(x[-w:].cpu() for x in (q, k, v)), g, d ** -0.5)
    mo, mf = reference(*(x[-w:].cpu().abs() for x in (q, k, v)), g, d ** -0.5)
    assert ((out[-100:].double().cpu() - eo[-100:]).abs() <= 2.0 ** -10 * mo[-100:] + 1e-4).all()
    assert ((final.double().cpu() - ef).abs() <= 2.0 ** -14 * mf).all()


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
def test_offsets_past_32_bits(clef, dtype):
    """Token strides of 2^23 elements: 600 tokens reach past 2^32."""
    T, H, d, stride = 600, 1, 64, 1 << 23
    if torch.cuda.mem_get_info()[0] < 32 << 30:
        pytest.skip("needs 32 GiB of device memory")
    q, k, v = _inputs(8, T, H, H, d, d, dtype)
    flat = torch.empty((T - 1) * stride + 4 * d, dtype=dtype, device="cuda")
    views = [torch.as_strided(flat, (T, H, d), (stride, d, 1), i * d) for i in range(4)]
    for x, y in zip(views, (q, k, v)):
        x.copy_(y)
    g = _slopes(H)
    _, final = clef.LinearScan(d, d).prefill(*views[:3], g.cuda(), out=views[3])
    check(views[3], final, q, k, v, g, d ** -0.5)


# ---------------------------------------------------------------------------- single tokens
def step_reference(kind, q, k, v, g, beta, slots, states, new, scale):
    """Row after row; returns (out of the live rows, new states, and both over absolute values)."""
    Hv = v.shape[1]
    rep = Hv // q.shape[1]
    out = torch.full(v.shape, float("nan"), dtype=torch.float64)
    mout, new, mnew = out.clone(), new.double().clone(), new.double().abs().clone()
    seen = set()
    for b in range(q.shape[0]):
        slot = b if slots is None else int(slots[b])
        if not 0 <= slot < new.shape[0]:
            continue
        if slot in seen:
            s, m = new[slot], mnew[slot]
        else:
            s = torch.zeros_like(new[0]) if states is None else (states if states.dim() == 3 else states[slot]).double()
            m = s.abs()
        seen.add(slot)
        qq, kk = (x[b].double().repeat_interleave(rep, 0) for x in (q, k))
        vv = v[b].double()
        if kind == "delta":
            qq = qq / (qq.square().sum(1, keepdim=True) + 1e-6).sqrt()
            kk = kk / (kk.square().sum(1, keepdim=True) + 1e-6).sqrt()
            s, m = (x * torch.exp(g[b].double())[:, None, None] for x in (s, m))
            bb = beta[b].double()[:, None]
            d = (vv - (kk[:, :, None] * s).sum(1)) * bb
            md = (vv.abs() + (kk.abs()[:, :, None] * m).sum(1)) * bb
        else:
            s, m = (x * _power(g, torch.tensor([1]))[..., None] for x in (s, m))
            d, md = vv, vv.abs()
        new[slot] = s + kk[:, :, None] * d[:, None, :]
        mnew[slot] = m + kk.abs()[:, :, None] * md[:, None, :]
        out[b] = scale * (qq[:, :, None] * new[slot]).sum(1)
        mout[b] = abs(scale) * (qq.abs()[:, :, None] * mnew[slot]).sum(1)
    return out, new, mout, mnew


def run_step(clef, kind, dtype, B, Hk, Hv, dk, dv, slots=None, nslots=None, states="pool", in_place=False, seed=0,
             out_dtype=None, gates=F32):
    nslots = nslots or B
    q, k, v = _inputs(seed, B, Hk, Hv, dk, dv, dtype)
    beta = torch.sigmoid(_randn(seed + 7, B, Hv)).to(gates)
    g = _slopes(Hv) if kind == "linear" else (-_randn(seed + 8, B, Hv).abs()).to(gates)
    old = {"pool": _randn(seed + 9, nslots, Hv, dk, dv), "one": _randn(seed + 9, Hv, dk, dv), "none": None}[states]
    new = old if in_place else _randn(seed + 10, nslots, Hv, dk, dv)
    out_dtype = out_dtype or dtype
    cout = torch.full((B, Hv, dv), 7.0, dtype=out_dtype, device="cuda")
    cq, ck, cv, cg, cb, cold = _cuda(q, k, v, g, beta, old)
    cnew = cold if in_place else new.cuda()
    cslots = None if slots is None else torch.tensor(slots, dtype=torch.int32, device="cuda")
    scan = clef.DeltaScan(dk, dv) if kind == "delta" else clef.LinearScan(dk, dv)
    args = (cq, ck, cv, cg) + ((cb,) if kind == "delta" else ()) + (cold,)
    got = scan.step(*args, slots=cslots, new_states=None if in_place else cnew, out=cout)
    assert got is cout
    eo, en, mo, mn = step_reference(kind, q, k, v, g, beta, slots, old, new, dk ** -0.5)
    live = torch.isfinite(eo[:, 0, 0])
    out = cout.double().cpu()
    assert (out[~live] == 7.0).all()
    # an output: sums over dk rows, twice in the delta rule (d, then o), of at most five rounded factors;
    # expf, sqrt and the division are within 2 units of theirs.  Repeated rows add theirs.
    rows = 1 if slots is None else max(slots.count(x) for x in slots)
    sums = (2 * dk + 24) * rows * 2.0 ** -24
    bound = sums * mo + (2.0 ** -11 * eo.abs() + 2.0 ** -25 if out_dtype == F16 else 0.0)
    err = (out - eo).abs()[live]
    assert (err <= bound[live]).all(), f"out: {float((err / bound[live]).max()):.3g} of the bound"
    named = torch.zeros(nslots, dtype=torch.bool)
    for b in range(B):
        s = b if slots is None else slots[b]
        if 0 <= s < nslots:
            named[s] = True
    cn = cnew.double().cpu()
    assert torch.equal(cn[~named], new.double()[~named])
    err = (cn - en).abs()[named]
    assert (err <= sums * mn[named]).all(), f"state: {float((err / (sums * mn[named])).max()):.3g} of the bound"


STEPS = [(1, 1, 1, 1, 1), (1, 16, 32, 128, 128), (3, 2, 6, 100, 72), (5, 1, 5, 128, 13), (2, 4, 4, 64, 64),
         (17, 16, 32, 128, 128), (33, 2, 2, 40, 24), (9, 1, 1, 128, 100), (7, 8, 8, 127, 128)]


@gpu
@pytest.mark.parametrize("kind", ["delta", "linear"])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("B,Hk,Hv,dk,dv", STEPS)
def test_step(clef, B, Hk, Hv, dk, dv, dtype, kind):
    run_step(clef, kind, dtype, B, Hk, Hv, dk, dv, seed=B)
    run_step(clef, kind, dtype, B, Hk, Hv, dk, dv, seed=B, in_place=True)


@gpu
@pytest.mark.parametrize("kind", ["delta", "linear"])
@pytest.mark.parametrize("states", ["pool", "one", "none"])
def test_step_slots(clef, states, kind):
    """A pool larger than the batch, rows without a request, and one state for all."""
    slots = [4, -1, 0, 9, 7, 100, 2 ** 31 - 1, -2 ** 31, 3]
    run_step(clef, kind, F16, len(slots), 2, 4, 64, 64, slots=slots, nslots=11, states=states, out_dtype=F32)
    if states == "pool":
        run_step(clef, kind, F32, len(slots), 2, 4, 64, 64, slots=slots, nslots=11, in_place=True, gates=F16)


@gpu
@pytest.mark.parametrize("kind", ["delta", "linear"])
@pytest.mark.parametrize("in_place", [True, False])
def test_step_rows_of_one_request(clef, in_place, kind):
    """Rows that share a slot are its tokens in row order."""
    run_step(clef, kind, F32, 10, 2, 4, 128, 128, slots=[1, 0, 1, 1, -1, 2, 0, 1, 5, 5], nslots=6, in_place=in_place)
    many = [i % 3 for i in range(300)]
    run_step(clef, kind, F16, 300, 1, 1, 32, 16, slots=many, nslots=4, in_place=in_place, out_dtype=F32)


@gpu
@pytest.mark.parametrize("kind", ["delta", "linear"])
def test_step_many_rows(clef, kind):
    run_step(clef, kind, F16, 1500, 1, 1, 16, 8)
    run_step(clef, kind, F16, 600, 1, 2, 128, 128, slots=[(7 * i) % 601 for i in range(600)], nslots=601)


@gpu
@pytest.mark.parametrize("kind", ["delta", "linear"])
def test_step_pool_past_32_bits(clef, kind):
    """States behind 2^31 elements of the pool, in place."""
    Hv, d, n = 32, 128, 4098
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GiB of device memory")
    pool = torch.empty((n, Hv, d, d), device="cuda")
    slots = [n - 1, 5, n - 2]
    old = _randn(1, 3, Hv, d, d)
    for i, s in enumerate(slots):
        pool[s] = old[i].cuda()
    q, k, v = _inputs(3, 3, 16, Hv, d, d, F32)
    g = _slopes(Hv) if kind == "linear" else -_randn(8, 3, Hv).abs()
    beta = torch.sigmoid(_randn(7, 3, Hv))
    scan = clef.DeltaScan(d, d) if kind == "delta" else clef.LinearScan(d, d)
    args = _cuda(q, k, v, g) + ([beta.cuda()] if kind == "delta" else [])
    out = scan.step(*args, pool, slots=torch.tensor(slots, dtype=torch.int32, device="cuda"))
    eo, en, mo, mn = step_reference(kind, q, k, v, g, beta, None, old, old, d ** -0.5)
    sums = (2 * d + 24) * 2.0 ** -24
    assert ((out.double().cpu() - eo).abs() <= sums * mo).all()
    for i, s in enumerate(slots):
        assert ((pool[s].double().cpu() - en[i]).abs() <= sums * mn[i]).all()


@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
def test_steps_continue_a_prompt(clef, dtype):
    """Tokens one by one from a prompt's state give what the prompt with them gives."""
    T, n, Hk, Hv, d = 90, 6, 2, 4, 64
    q, k, v = _inputs(2, T + n, Hk, Hv, d, d, dtype)
    g = _slopes(Hv)
    scan = clef.LinearScan(d, d)
    cq, ck, cv, cg = _cuda(q, k, v, g)
    out, state = scan.prefill(cq[:T], ck[:T], cv[:T], cg)
    outs = [out] + [scan.step(cq[t:t + 1], ck[t:t + 1], cv[t:t + 1], cg, state[None]) for t in range(T, T + n)]
    check(torch.cat(outs), state, q, k, v, g, scan.scale)


@gpu
def test_delta_steps_continue_the_scan(clef):
    """The DeltaNet step from the scan's captured state against the scan itself (strict profile's bar)."""
    import workloads
    T, n, H, d = 130, 5, 4, 64
    q, k, v, g, beta = workloads.scan_inputs(3, T + n, H, H, d, d)
    scan = clef.DeltaScan(d, d, "strict")
    out, mid, final = scan.prefill(q, k, v, g, beta, capture=T)
    state = mid[None].clone()
    for t in range(T, T + n):
        o = scan.step(*(x[t:t + 1] for x in (q, k, v, g, beta)), state)
        assert torch.allclose(o[0], out[t], rtol=1e-4, atol=1e-5)
    assert torch.allclose(state[0], final, rtol=1e-4, atol=1e-5)


# ---------------------------------------------------------------------------- streams and graphs
@gpu
def test_captured_graph_replays(clef):
    """Prompt, ragged prompt and steps in one graph, replayed on changed inputs between eager calls."""
    lens, H, d = [200, 0, 333, 64], 2, 64
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    T = int(cu[-1])
    q, k, v = _cuda(*_inputs(0, T, H, H, d, d, F16))
    g = _slopes(H).cuda()
    slots = torch.tensor([2, 0, -1, 2], dtype=torch.int32, device="cuda")
    scan = clef.LinearScan(d, d)

    def work(pool, row):
        a, fa = scan.prefill(q, k, v, g)
        b, fb = scan.prefill_varlen(q, k, v, g, cu, initial=fa)
        c = scan.step(q[:4], k[:4], v[:4], g, pool, slots=slots, out=row)
        return a, b, fb, c, pool

    row = torch.zeros((4, H, d), device="cuda")
    pool = torch.zeros((4, H, d, d), device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work(pool, row)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work(pool, row)
    for i in range(4):
        for x, y in zip((q, k, v), _inputs(100 + i, T, H, H, d, d, F16)):
            x.copy_(y)
        if i == 2:  # other lengths, the same launch
            cu.copy_(torch.tensor([0, 64, 65, 500, T - 5], dtype=torch.int32))
        pool.copy_(_randn(i, 4, H, d, d))
        row.zero_()
        again_pool, again_row = pool.clone(), row.clone()
        eager = work(again_pool, again_row)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        n = T - 5 if i >= 2 else T
        for x, y in zip(outs, eager):
            m = n if x.shape[0] == T else x.shape[0]
            assert torch.equal(x[:m], y[:m]), f"replay {i}"


@gpu
def test_two_streams_at_once(clef):
    T, H, d = 700, 2, 128
    a, b = _cuda(*_inputs(0, T, H, H, d, d, F16)), _cuda(*_inputs(5, T, H, H, d, d, F32))
    g = _slopes(H).cuda()
    scan = clef.LinearScan(d, d)
    want = [scan.prefill(*x, g) for x in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, x in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(scan.prefill(*x, g))
    torch.cuda.synchronize()
    for i in range(2):
        for o, f in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(f, want[i][1])
