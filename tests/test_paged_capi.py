"""Refusals of the paged cache's entry points: each bad call is turned down on the
host, before any launch (no GPU here)."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def clef():
    import clef_hip
    clef_hip.lib()
    return clef_hip


KEEP = []


def cache(clef, **kw):
    a = dict(k=1 << 20, vt=1 << 21, k_stride=0, vt_stride=0, num_pages=9, page=32, kv_heads=2, d=64, dtype=1)
    assert set(kw) <= set(a)
    a.update(kw)
    KEEP.append(clef.PagedCacheDesc(*a.values()))
    return C.addressof(KEEP[-1])


CACHE = [dict(k=None), dict(vt=None), dict(k=(1 << 20) + 8), dict(vt=(1 << 21) + 2), dict(k_stride=4095),
         dict(vt_stride=4088), dict(k_stride=4097), dict(vt_stride=4100), dict(k_stride=-8), dict(num_pages=0),
         dict(num_pages=-1), dict(page=0), dict(page=8), dict(page=48), dict(page=512), dict(page=-32),
         dict(kv_heads=0), dict(kv_heads=3), dict(kv_heads=257), dict(d=0), dict(d=60), dict(d=264), dict(dtype=2)]
BATCH = [dict(cache=None), dict(table=None), dict(width=0), dict(width=-1), dict(width=(1 << 19) + 1), dict(cu=None),
         dict(lens=None), dict(nseq=0), dict(nseq=4097), dict(T=0), dict(T=65537), dict(heads=0), dict(heads=257),
         dict(heads=7)]


def args(clef, kind, kw):
    desc = {k[6:]: v for k, v in kw.items() if k.startswith("cache_")}
    a = dict(cache=cache(clef, **desc), table=256, width=5, cu=256, lens=256, nseq=3, T=9)
    a.update({
        "append": dict(q=256, ldq=0, hsq=0, k=256, ldk=0, v=256, ldv=0, heads=8, qn=256, kn=256, eps=1e-6, pos=256,
                       ldpos=9, axes=3, axis_of=bytes([0, 1, 2, 0] * 4), rot=32, theta=1e7, out=256, ldo=9),
        "attention": dict(q=256, ldq=9, heads=8, gate=256, ldg=512, hsg=64, window=0, sinks=0, y=256, ldy=512,
                          lse=256, ws=256, wsb=1 << 40),
        "weights": dict(q=256, ldq=9, heads=8, lse=256, window=0, sinks=0, scores=256, new=256, ws=256, wsb=1 << 40)}[kind])
    kw = {k: v for k, v in kw.items() if not k.startswith("cache_")}
    assert set(kw) <= set(a), kw
    a.update(kw)
    return tuple(a.values()) + (None,)


OWN = {
    "append": [dict(q=None), dict(k=None), dict(v=None), dict(qn=None), dict(kn=None), dict(out=None), dict(ldq=511),
               dict(hsq=63), dict(ldk=127), dict(ldv=127), dict(ldo=8), dict(rot=33), dict(rot=-2), dict(rot=66),
               dict(theta=0.0), dict(theta=float("nan")), dict(theta=float("inf")), dict(eps=-1.0),
               dict(eps=float("nan")), dict(axes=0), dict(axes=5), dict(axes=2), dict(ldpos=8), dict(out=264)],
    "attention": [dict(q=None), dict(gate=None), dict(y=None), dict(ws=None), dict(wsb=0), dict(ws=264), dict(ldq=8), dict(ldq=(1 << 22) + 1),
                  dict(ldg=511), dict(hsg=63), dict(ldy=511), dict(window=-1), dict(window=(1 << 24) + 1),
                  dict(sinks=-1), dict(sinks=(1 << 24) + 1), dict(q=264)],
    "weights": [dict(q=None), dict(lse=None), dict(scores=None), dict(new=None), dict(ldq=8), dict(window=-1),
                dict(window=(1 << 24) + 1), dict(sinks=-1), dict(sinks=(1 << 24) + 1), dict(q=264), dict(ws=264), dict(ldq=(1 << 22) + 1), dict(T=900, ldq=900, ws=None),
                dict(T=900, ldq=900, wsb=0)],
}
NAME = {"append": "clef_paged_append", "attention": "clef_attention_gated_paged", "weights": "clef_paged_weights"}


@pytest.mark.parametrize("kind,bad", [(k, b) for k in OWN for b in
                                      OWN[k] + BATCH + [{"cache_" + n: v for n, v in c.items()} for c in CACHE]],
                         ids=str)
def test_batches_refuse(clef, kind, bad):
    assert getattr(clef.lib(), NAME[kind])(*args(clef, kind, bad)) < 0
    assert "paged " + kind in clef.last_error()


@pytest.mark.parametrize("kind", ["attention", "weights"])
def test_workspace(clef, kind):
    L = clef.lib()
    size = {"attention": L.clef_attention_paged_workspace, "weights": L.clef_paged_weights_workspace}[kind]
    good = (900, 3, 5, 32, 1, 8, 2, 64)
    n = size(*good)
    assert n > 256 and n % 256 == 0
    assert getattr(L, NAME[kind])(*args(clef, kind, dict(T=900, ldq=900, wsb=n - 1))) < 0
    for i, bad in ((0, 0), (0, 65537), (1, 0), (1, 4097), (2, 0), (2, (1 << 19) + 1), (3, 24), (4, 3), (5, 0), (5, 7),
                   (6, 0), (7, 4), (7, 264)):
        a = list(good)
        a[i] = bad
        assert size(*a) == 0, (i, bad)
    # the largest call that is allowed
    assert size(65536, 4096, 1 << 20, 16, 0, 256, 256, 256) > 0


def evict(clef, **kw):
    desc, to = ({k[len(n):]: v for k, v in kw.items() if k.startswith(n)} for n in ("cache_", "to_cache_"))
    a = dict(cache=cache(clef, **desc), table=256, width=5, lens=256, nseq=3, scores=256, budget=70, sinks=4, recent=8,
             to=cache(clef, **{"k": 1 << 22, "vt": 1 << 23, **to}), to_table=256, to_width=3, to_scores=256, new=256,
             keep=256)
    kw = {k: v for k, v in kw.items() if not k.startswith(("cache_", "to_cache_"))}
    assert set(kw) <= set(a), kw
    a.update(kw)
    return tuple(a.values()) + (None,)


@pytest.mark.parametrize("bad", [
    dict(cache=None), dict(to=None), dict(table=None), dict(to_table=None), dict(lens=None), dict(scores=None),
    dict(scores=264), dict(to_scores=None), dict(new=None), dict(keep=None), dict(width=0), dict(to_width=0), dict(nseq=0),
    dict(nseq=4097), dict(budget=0), dict(budget=-1), dict(budget=11), dict(budget=97), dict(sinks=-1),
    dict(sinks=71), dict(recent=-1), dict(recent=67), dict(sinks=2 ** 31 - 1), dict(recent=2 ** 31 - 1),
    dict(to_cache_page=16, to_width=6), dict(to_cache_kv_heads=1), dict(to_cache_d=72), dict(to_cache_dtype=0)] +
    [{n + "cache_" + k: v for k, v in c.items()} for c in CACHE for n in ("", "to_")
     if c not in (dict(kv_heads=3), dict(kv_heads=257))], ids=str)
def test_evict_refuses(clef, bad):
    assert clef.lib().clef_paged_evict(*evict(clef, **bad)) < 0
    assert "paged evict" in clef.last_error()


def test_evict_refuses_more_than_a_launch(clef):
    assert clef.lib().clef_paged_evict(*evict(clef, nseq=4096, width=1 << 19, to_width=1 << 19, budget=1 << 24)) < 0


def test_binding_refuses_host_tensors_and_shapes(clef):
    import torch
    k, vt = torch.zeros((5, 2, 16, 8)), torch.zeros((5, 2, 8, 16))
    for bad in ((k[0], vt), (k, k), (k.half(), vt), (k.transpose(2, 3), vt), (k[:, :1], vt),
                (k[:, :, ::2], vt[:, :, :, ::2]), (k.double(), vt.double()), (k[:1].expand(5, -1, -1, -1), vt)):
        with pytest.raises(clef.ClefError):
            clef.PagedCache(*bad)
    c = clef.PagedCache(k, vt)
    cu, lens, pages = torch.tensor([0, 3], dtype=torch.int32), torch.tensor([3], dtype=torch.int32), \
        torch.zeros((1, 2), dtype=torch.int32)
    q, gate, w = torch.zeros((4, 3, 8)), torch.zeros((3, 4, 8)), torch.ones(8)
    lse, scores = torch.zeros((3, 4)), torch.zeros((5, 2, 16))
    x, kv = torch.zeros((3, 4, 8)), torch.zeros((3, 2, 8))
    calls = [
        (c.attention_gated, [(q, gate, cu, lens, pages), (q.half(), gate, cu, lens, pages),
                             (q[:, :, :4], gate, cu, lens, pages), (q, gate[:2], cu, lens, pages),
                             (q, gate, cu.long(), lens, pages), (q, gate, cu, lens.float(), pages),
                             (q, gate, cu, lens, pages[0]), (q, gate, cu, lens, pages.long())]),
        (c.add_weights, [(q, lse, cu, lens, pages, scores), (q, lse[:2], cu, lens, pages, scores),
                         (q, lse, cu, lens, pages, scores[:4]), (q, lse.half(), cu, lens, pages, scores),
                         (q, lse, cu, lens, pages, scores.double())]),
        (c.append, [(x, kv, kv, w, w, cu, lens, pages, 8, 1e4), (x, kv[:2], kv, w, w, cu, lens, pages, 8, 1e4),
                    (x, kv, kv.half(), w, w, cu, lens, pages, 8, 1e4), (x, kv, kv, w[:4], w, cu, lens, pages, 8, 1e4),
                    (x, kv, kv, w, w, cu, lens, pages, 8, 1e4, cu), (x, kv, kv, w, w, cu, lens, pages, 8, 1e4, None, [0]),
                    (x, kv, kv, w, w, cu, lens, pages, 8, 1e4, None, [0, 0, 0, 1]),
                    (x.expand(3, 4, 8)[:, :1].expand(3, 4, 8), kv, kv, w, w, cu, lens, pages, 8, 1e4)]),
        (c.evict, [(scores, lens, pages, 4, c, pages, scores), (scores[:3], lens, pages, 4, c, pages, scores),
                   (scores, lens, pages[:0], 4, c, pages, scores), (scores, lens, pages, 0, c, pages, scores)])]
    for call, several in calls:
        for a in several:
            with pytest.raises(clef.ClefError):
                call(*a)


def test_evict_refuses_lengths_that_overlap(clef):
    for lens, new in ((256, 260), (260, 256), (256, 264), (264, 256)):
        assert clef.lib().clef_paged_evict(*evict(clef, lens=lens, new=new)) < 0
        assert "new_lens" in clef.last_error()
