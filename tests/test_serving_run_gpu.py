"""The operators together, as a batch of requests runs through a hybrid stack: a
shared prefix is taken once (scan, linear attention, keys and values), every
request is forked from its states, and tokens follow one by one (DeltaNet step,
linear-attention step, shared-prefix attention on growing caches).  Each layer's
outputs equal those of its prompt form over the same tokens at once.

Bounds.  DeltaNet: the strict profile's bar.  Linear attention: the step is f32 and the
f16 prompt form rounds one factor of each product once (2^-11 of it; f32 sums add less
than 2^-13), so the two differ by at most (2^-11 + 2^-13) M, with M the same output over
absolute values, which the step itself gives on |q|, |k|, |v| and the state of those.
Attention: each form rounds the weights once (2^-11 of them) and its output; the prompt
form also the attention and the gate: at most 2 2^-11 max |v| + 4 2^-11 |y|."""
import pytest
import torch

gpu = pytest.mark.gpu

HEADS, KVH, D, ROT, THETA = 8, 2, 64, 32, 10000.0
HK, HV, W = 2, 4, 64


@pytest.fixture(scope="module")
def clef():
    import clef_hip
    clef_hip.lib()
    return clef_hip


def _randn(gen, *shape, dtype=torch.float16):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


@gpu
@pytest.mark.parametrize("prefix", [72, 520])
def test_requests_behind_one_prefix(clef, prefix):
    lens = [5, 1, 7, 3]  # tokens of each request behind the prefix
    n, steps, room = len(lens), max(lens), 16
    gen = torch.Generator(device="cuda").manual_seed(prefix)
    total = sum(lens)
    cu = [sum(lens[:i]) for i in range(n + 1)]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    every = prefix + total  # all tokens: the prefix, then the requests' packed

    # ---- linear layers: q, k, v of every token
    q, k = (_randn(gen, every, HK, W) for _ in range(2))
    v = _randn(gen, every, HV, W)
    g = -torch.rand((every, HV), generator=gen, device="cuda")
    beta = torch.rand((every, HV), generator=gen, device="cuda")
    slopes = -torch.exp2(-8.0 * torch.arange(1, HV + 1, device="cuda") / HV)
    delta, linear = clef.DeltaScan(W, W, "strict"), clef.LinearScan(W, W)
    head = slice(0, prefix)
    _, _, delta_state = delta.prefill(q[head], k[head], v[head], g[head], beta[head])
    _, linear_state = linear.prefill(q[head], k[head], v[head], slopes)
    tail = slice(prefix, every)
    want_delta, final_delta = delta.prefill_varlen(q[tail], k[tail], v[tail], g[tail], beta[tail], ints(cu),
                                                   initial=delta_state)
    want_linear, final_linear = linear.prefill_varlen(q[tail], k[tail], v[tail], slopes, ints(cu),
                                                      initial=linear_state)

    # the same over absolute values
    aqs, aks, avs = q.abs(), k.abs(), v.abs()
    _, abs_state = linear.prefill(aqs[head], aks[head], avs[head], slopes)
    abs_pool = torch.zeros((n, HV, W, W), device="cuda")

    # ---- attention layer: raw projections, norm and rotary as the backbone applies them
    aq, ak, av = _randn(gen, every, HEADS * D), _randn(gen, every, KVH * D), _randn(gen, every, KVH * D)
    gate = _randn(gen, every, HEADS, D)
    norm = torch.ones(D, device="cuda")
    keys = clef.qk_norm_rotary(ak[head], KVH, D, norm, ROT, THETA)
    values = clef.values_transposed(av[head], KVH, D)
    rotated = lambda x, heads: clef.qk_norm_rotary_varlen(x, heads, D, norm, ROT, THETA, ints(cu), pos0=prefix)  # noqa: E731
    tail_q, tail_k = rotated(aq[tail], HEADS), rotated(ak[tail], KVH)
    want = clef.attention_gated_varlen(tail_q, tail_k, clef.values_transposed(av[tail], KVH, D), gate[tail], ints(cu),
                                       prefix_k=keys, prefix_vt=values)

    # ---- token by token: row s of a step is request s's next token, empty once it has none
    pools = [torch.full((n, HV, W, W), float("nan"), device="cuda") for _ in range(2)]
    cache_k = torch.zeros((KVH, n * room, D), dtype=torch.float16, device="cuda")
    cache_v = torch.zeros((KVH, D, n * room), dtype=torch.float16, device="cuda")
    starts = ints([s * room for s in range(n)])
    for i in range(steps):
        live = [s for s in range(n) if i < lens[s]]
        rows = torch.tensor([prefix + cu[s] + i if s in live else 0 for s in range(n)], device="cuda")
        slots = ints([s if s in live else -1 for s in range(n)])
        x = [t[rows] for t in (q, k, v, g, beta)]
        # the first step reads the prefix's state for every request, the others their own
        states = (delta_state, linear_state) if i == 0 else pools
        got_delta = delta.step(*x, states[0], slots=slots, new_states=pools[0])
        got_linear = linear.step(x[0], x[1], x[2], slopes, states[1], slots=slots, new_states=pools[1])
        most = linear.step(aqs[rows], aks[rows], avs[rows], slopes, abs_state if i == 0 else abs_pool, slots=slots,
                           new_states=abs_pool)
        for s in live:
            cache_k[:, s * room + i] = tail_k[:, cu[s] + i]
            cache_v[:, :, s * room + i] = av[prefix + cu[s] + i].view(KVH, D)
        step_q = torch.stack([tail_q[:, cu[s] + i] if s in live else torch.zeros_like(tail_q[:, 0])
                              for s in range(n)], 1).contiguous()
        cut = [0]
        for s in range(n):
            cut.append(cut[-1] + (s in live))
        packed = step_q[:, live].contiguous()
        y = clef.attention_gated_shared(packed, cache_k, cache_v, gate[rows[live]], ints(cut), starts,
                                        ints([min(i + 1, m) for m in lens]), prefix_k=keys, prefix_vt=values,
                                        max_keys=room)
        for j, s in enumerate(live):
            t = cu[s] + i
            assert torch.allclose(got_delta[s], want_delta[t], rtol=1e-4, atol=1e-5)
            assert ((got_linear[s] - want_linear[t]).abs() <= (2.0 ** -11 + 2.0 ** -13) * most[s]).all()
            assert torch.allclose(y[j].float(), want[t].float(), rtol=2.0 ** -9, atol=2.0 ** -10 * float(av.abs().max()))
    assert torch.allclose(pools[0], final_delta, rtol=1e-4, atol=1e-5)
    # states: f32 sums, and the prompt form's factors held to 22 bits
    assert ((pools[1] - final_linear).abs() <= 2.0 ** -13 * abs_pool).all()
