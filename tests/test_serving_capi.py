"""Refusals of the linear-attention, step and shared-prefix attention entry points:
each bad call is turned down on the host, before any launch (no GPU here)."""
import pytest


@pytest.fixture(scope="module")
def L():
    import clef_hip
    return clef_hip.lib()


def scan(**kw):
    a = dict(q=256, k=256, v=256, sqk=0, sv=0, dt=1, g=256, cu=256, nseq=3, T=100, Hk=2, Hv=4, dk=64, dv=64, scale=0.125,
             initial=None, stride=0, out=256, so=0, dto=1, final=None, ws=256, wsb=1 << 40)
    assert set(kw) <= set(a)
    a.update(kw)
    return tuple(a.values()) + (None,)


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(k=None), dict(v=None), dict(g=None), dict(out=None), dict(cu=None), dict(T=3000, ws=None),
    dict(T=3000, wsb=0), dict(ws=257), dict(T=0), dict(T=(1 << 20) + 1), dict(nseq=0), dict(nseq=4097), dict(Hk=0), dict(Hk=3), dict(Hv=257),
    dict(dk=0), dict(dk=129), dict(dv=0), dict(dv=129), dict(dt=2), dict(dto=2), dict(sqk=127), dict(sv=255),
    dict(so=255), dict(stride=-1), dict(stride=4 * 64 * 64 - 1), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(initial=1 << 20, stride=4 * 64 * 64, final=(1 << 20) + 64)], ids=str)
def test_linear_scan_refuses(L, bad):
    import clef_hip
    assert L.clef_linear_scan_varlen(*scan(**bad)) < 0
    assert "linear attention scan" in clef_hip.last_error()


def test_linear_scan_workspace(L):
    assert L.clef_linear_scan_workspace(0, 1, 1, 1, 64, 64, 1) == 0
    assert L.clef_linear_scan_workspace(10, 0, 1, 1, 64, 64, 1) == 0
    assert L.clef_linear_scan_workspace(10, 1, 2, 3, 64, 64, 1) == 0
    assert L.clef_linear_scan_workspace(10, 1, 1, 1, 64, 64, 3) == 0
    n = L.clef_linear_scan_workspace(3000, 3, 2, 4, 64, 64, 1)
    assert n > 256 and L.clef_linear_scan_varlen(*scan(T=3000, wsb=n - 1)) < 0
    assert L.clef_linear_scan_workspace(1 << 20, 4096, 1, 2, 128, 128, 0) % 256 == 0


def step(kind, **kw):
    a = dict(q=256, k=256, v=256, sqk=0, sv=0, dt=1, g=256)
    if kind == "delta":
        a.update(beta=256, sgb=0, dtg=0)
    a.update(slots=256, B=5, Hk=2, Hv=4, dk=64, dv=64)
    if kind == "linear":
        a.update(scale=0.125)
    a.update(states=1 << 20, stride=4 * 64 * 64, new=1 << 30, nslots=7, out=256, so=0, dto=1)
    assert set(kw) <= set(a)
    a.update(kw)
    return tuple(a.values()) + (None,)


COMMON = [dict(q=None), dict(k=None), dict(v=None), dict(g=None), dict(new=None), dict(out=None), dict(B=0),
          dict(B=4097), dict(Hk=0), dict(Hk=3), dict(Hv=257), dict(dk=0), dict(dk=129), dict(dv=0), dict(dv=129),
          dict(dt=2), dict(dto=5), dict(sqk=127), dict(sv=255), dict(so=255), dict(nslots=0),
          dict(slots=None, nslots=4), dict(stride=-1), dict(stride=4 * 64 * 64 - 1),
          dict(new=(1 << 20) + 4 * 64), dict(states=1 << 20, new=1 << 20, stride=0),
          dict(states=1 << 20, new=1 << 20, stride=4 * 64 * 64 + 4)]


@pytest.mark.parametrize("kind,bad", [("linear", b) for b in COMMON + [dict(scale=float("nan"))]] +
                         [("delta", b) for b in COMMON + [dict(beta=None), dict(sgb=3), dict(dtg=7)]], ids=str)
def test_steps_refuse(L, kind, bad):
    import clef_hip
    fn = L.clef_linear_step if kind == "linear" else L.clef_delta_step
    assert fn(*step(kind, **bad)) < 0
    assert "step" in clef_hip.last_error()


def shared(**kw):
    a = dict(q=256, ldq=9, pk=256, ldpk=1000, pvt=256, ldpv=1000, np=999, k=256, ldk=300, vt=256, ldv=304, cu=256,
             starts=256, lens=256, nseq=4, T=9, max_keys=50, dt=1, heads=8, kvh=2, d=64, gate=256, ldg=512, hsg=64,
             y=256, ldy=512, ws=256, wsb=1 << 40)
    assert set(kw) <= set(a)
    a.update(kw)
    return tuple(a.values()) + (None,)


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(gate=None), dict(y=None), dict(cu=None), dict(pk=None), dict(pvt=None), dict(k=None),
    dict(vt=None), dict(starts=None), dict(lens=None), dict(ws=None), dict(wsb=0), dict(ws=264), dict(ldq=8),
    dict(ldpk=998), dict(ldpv=992), dict(ldpv=1001), dict(ldv=303), dict(ldk=0), dict(ldv=0), dict(ldk=1 << 31),
    dict(ldv=1 << 31), dict(nseq=0), dict(nseq=4097), dict(T=0), dict(T=65537), dict(np=-1), dict(np=(1 << 24) + 1),
    dict(max_keys=-1), dict(max_keys=(1 << 24) + 1), dict(np=0, max_keys=0), dict(dt=2), dict(heads=0), dict(heads=257),
    dict(kvh=0), dict(kvh=3), dict(d=0), dict(d=60), dict(d=264), dict(hsg=63), dict(ldg=511), dict(ldy=511),
    dict(q=264), dict(pk=264), dict(pvt=258), dict(k=260), dict(vt=264)], ids=str)
def test_shared_attention_refuses(L, bad):
    import clef_hip
    assert L.clef_attention_gated_shared(*shared(**bad)) < 0
    assert "shared-prefix attention" in clef_hip.last_error()


@pytest.mark.parametrize("bad", [dict(ldk=(1 << 30) + 1), dict(ldv=(1 << 30) + 8)], ids=str)
def test_shared_attention_refuses_rows_past_its_block_numbers(L, bad):
    """Blocks of keys are numbered with 32 bits, a step of the waves behind the last one included."""
    assert L.clef_attention_gated_shared(*shared(**bad)) < 0


def test_shared_attention_workspace(L):
    assert L.clef_attention_shared_workspace(0, 1, 8, 8, 1, 8, 2, 64) == 0
    assert L.clef_attention_shared_workspace(4, 1, 0, 0, 1, 8, 2, 64) == 0
    assert L.clef_attention_shared_workspace(4, 1, 8, 8, 1, 8, 2, 65) == 0
    n = L.clef_attention_shared_workspace(9, 4, 999, 50, 1, 8, 2, 64)
    assert n > 256 and L.clef_attention_gated_shared(*shared(wsb=n - 1)) < 0


def test_binding_refuses_host_tensors_and_shapes():
    import torch

    import clef_hip as clef
    x, v, g = torch.zeros((3, 2, 8)), torch.zeros((3, 4, 8)), torch.zeros(4)
    scan = clef.LinearScan(8, 8)
    for args in ((x[:2], x, v, g), (x, x, v[:, :3], torch.zeros(4)), (x, x, v, torch.zeros(3)),
                 (x, x, v, g.double()), (x, x, v.half(), g), (x[:, 0], x[:, 0], v, g)):
        with pytest.raises(clef.ClefError):
            scan.prefill(*args)
    with pytest.raises(clef.ClefError):
        clef.LinearScan(8, 8).step(x, x, v, g, torch.zeros((3, 4, 8, 7)))
    with pytest.raises(clef.ClefError):
        clef.LinearScan(8, 8).step(x, x, v, g, torch.zeros((3, 4, 8, 8)), slots=torch.zeros(3))
    with pytest.raises(clef.ClefError):
        clef.LinearScan(8, 8).step(x, x, v, g, torch.zeros((3, 4, 8, 8)).double())
    with pytest.raises(clef.ClefError):
        clef.attention_gated_shared(torch.zeros((2, 3, 8)), None, None, torch.zeros((3, 2, 8)),
                                    torch.zeros(2, dtype=torch.int32), None, None)
