"""The device code of a paged cache's calls that finds requests and deals out work from
device tables (paged.hpp, paged_walk.hpp), compiled for the host with the threads of a
work-group as fibers (host_wave/): over tables that fit, every token and every block of
keys is found once, and over tables that do not, no index leaves its buffer."""
import ctypes as C
import pathlib
import subprocess

import numpy as np
import pytest

HERE = pathlib.Path(__file__).resolve().parent
CLANG = "/opt/rocm/llvm/bin/clang++"
INT_MIN, INT_MAX = -2 ** 31, 2 ** 31 - 1


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    out = tmp_path_factory.mktemp("host_wave") / "paged_tables.so"
    subprocess.run([CLANG, "-O1", "-std=c++17", "-fPIC", "-shared", "-I", str(HERE / "host_wave"), "-o", str(out),
                    str(HERE / "host_wave" / "paged_tables.cpp")], check=True)
    return C.CDLL(str(out))


def ints(x):
    return np.ascontiguousarray(np.clip(x, INT_MIN, INT_MAX).astype(np.int32))


def at(x):
    return x.ctypes.data_as(C.c_void_p)


def fitting(rng, nseq, T):
    """Offsets from 0, some requests empty, up to a few rows behind the last one."""
    total = int(rng.integers(0, T + 1))
    return np.concatenate([[0], np.sort(rng.integers(0, total + 1, nseq - 1)), [total]])


def bad(rng, nseq, T):
    kind = rng.integers(0, 5)
    if kind == 0:
        return rng.integers(INT_MIN, INT_MAX, nseq + 1, endpoint=True)
    if kind == 1:
        return rng.integers(-T, 2 * T + 1, nseq + 1)
    if kind == 2:
        return rng.integers(0, T + 1, nseq + 1)
    table = fitting(rng, nseq, T)
    if kind == 3:  # a fitting one with a few entries replaced
        table[rng.integers(0, nseq + 1, 3)] = rng.choice([INT_MIN, -1, 0, T // 2, T, T + 1, INT_MAX], 3)
        return table
    return table[::-1]


def requests(host, cu, lens, T, page, width, tokens):
    out = np.zeros((len(tokens), 4), np.int32)
    for i, t in enumerate(tokens):
        host.requests_at(at(cu), at(lens), len(lens), T, page, width, int(t), int(t) + 1, at(out[i:i + 1]))
    return out


# ---------------------------------------------------------------------------- requests
@pytest.mark.parametrize("nseq", [1, 2, 65, 4096])
def test_requests_stay_inside(host, nseq):
    """A request's tokens lie in the batch and its keys in its table, whatever the tables hold."""
    rng = np.random.default_rng(nseq)
    for i in range(30):
        T = int(rng.integers(1, 65537))
        cu, lens = bad(rng, nseq, T), rng.choice([INT_MIN, -1, 0, 1, 239, 240, 241, INT_MAX], nseq)
        if i == 0:
            cu[0], cu[1] = 1, INT_MIN
        cu, lens = ints(cu), ints(lens)
        out = np.zeros((nseq, 3), np.int32)
        host.requests_of(at(cu), at(lens), nseq, T, 16, 15, at(out))
        first, n, length = out.astype(np.int64).T
        assert (first == np.clip(cu[:-1], 0, T)).all()
        assert (n == np.maximum(np.clip(cu[1:], 0, T) - first, 0)).all()
        assert (length == np.clip(lens, 0, 240)).all()


# ---------------------------------------------------------------------------- the request of a token
@pytest.mark.parametrize("nseq", [1, 2, 63, 64, 65, 130, 4096])
def test_tokens_find_their_request(host, nseq):
    rng = np.random.default_rng(nseq)
    for _ in range(4):
        T = int(rng.integers(1, min(3 * nseq, 60000) + 2))
        cu = ints(fitting(rng, nseq, T))
        lens = ints(cu[1:] - cu[:-1] + rng.integers(0, 50, nseq))
        tokens = rng.integers(0, T, 40)
        for t, (s, first, n, length) in zip(tokens, requests(host, cu, lens, T, 16, 8192, tokens)):
            want = int(np.searchsorted(cu[1:], t, side="right"))
            assert s == (want if want < nseq else -1)
            if s >= 0:
                assert (first, n, length) == (cu[s], cu[s + 1] - cu[s], lens[s]) and first <= t < first + n




@pytest.mark.parametrize("nseq", [1, 2, 3, 63, 64, 65, 200, 4096])
def test_bad_tables_find_tokens_inside_a_request(host, nseq):
    """What a token's page is found by: its index among the request's keys is below their number,
    so the table's column is one of the request's."""
    rng = np.random.default_rng(nseq)
    special = [([0, 20, 3, 5], [5, 6, 240], 22), ([22, 22, 0, 0], [1, 2, INT_MAX], 22), ([0, 9, 2, 4], [9, 9, 240], 9)]
    for i in range(40):
        if nseq == 3 and i < len(special):
            cu, lens, T = special[i]
        else:
            T = int(rng.integers(1, 65537 if i % 2 else 300))
            cu, lens = bad(rng, nseq, T), rng.choice([INT_MIN, -1, 0, 1, 239, 240, 241, INT_MAX], nseq)
        cu, lens = ints(cu), ints(lens)
        tokens = range(T) if T <= 22 else rng.integers(0, T, 30)
        for t, (s, first, n, length) in zip(tokens, requests(host, cu, lens, T, 16, 15, tokens)):
            assert -1 <= s < nseq
            if s >= 0:
                assert 0 <= first <= t < first + int(n) <= T and 0 <= length <= 240
                assert length - n + (t - first) < 240  # max_pages * page


# ---------------------------------------------------------------------------- the line
PIECE = ("s", "kv", "tile", "b0", "b1", "head", "tail", "blocks", "rows", "first", "n", "last")


def pieces(host, cu, lens, T, page, width, kvh, G, R, cost, window, sinks, least, groups, threads, which=None, most=4000):
    """The pieces of each work-group, as dicts with its number on the line's order of groups."""
    out = np.zeros((most, len(PIECE)), np.int32)
    got = []
    for group in range(groups) if which is None else which:
        n = host.walk(at(cu), at(lens), len(lens), T, page, width, kvh, G, R, cost, window, sinks,
                      C.c_float(1.0 / (least * 64 * G)), group, groups, threads, at(out), most)
        assert n >= 0, "a request that there is not"
        got += [dict(zip(PIECE, row), group=group) for row in out[:n].tolist()]
    return got


def inside(y, nseq, T, kvh, groups):
    assert 0 <= y["s"] < nseq and 0 <= y["kv"] < kvh and y["tile"] >= 0 and y["rows"] > 0, y
    assert 0 <= y["b0"] <= y["b1"] <= y["blocks"], y
    assert 0 <= y["first"] and y["first"] + y["n"] <= T and y["last"] <= groups, y


@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4)])
@pytest.mark.parametrize("nseq,kvh,G,R,cost,threads", [(1, 2, 8, 256, 512, 512), (5, 2, 8, 16, 64, 256),
                                                       (70, 1, 3, 64, 64, 256), (600, 3, 1, 16, 64, 256)])
def test_every_block_is_dealt_once(host, nseq, kvh, G, R, cost, threads, window, sinks):
    rng = np.random.default_rng(nseq + window)
    groups, T = 64, 4 * nseq + 90
    cu = ints(fitting(rng, nseq, T))
    n = cu[1:] - cu[:-1]
    lens = ints(n + rng.integers(0, 700, nseq))
    got = pieces(host, cu, lens, T, 16, 400, kvh, G, R, cost, window, sinks, 2, groups, threads)
    tiles = {}
    for y in got:
        inside(y, nseq, T, kvh, groups)
        assert (y["first"], y["n"]) == (cu[y["s"]], n[y["s"]])
        tiles.setdefault((y["s"], y["kv"], y["tile"]), []).append(y)
    assert set(tiles) == {(s, kv, i) for s in range(nseq) for kv in range(kvh) for i in range(-(-int(n[s]) * G // R))}
    for parts in tiles.values():
        parts.sort(key=lambda y: (not y["head"], y["b0"]))
        assert parts[0]["head"] and parts[-1]["tail"]
        assert sum(y["head"] for y in parts) == sum(y["tail"] for y in parts) == 1
        assert parts[0]["b0"] == 0 and parts[-1]["b1"] == parts[-1]["blocks"]
        assert all(a["b1"] == b["b0"] for a, b in zip(parts, parts[1:]))


@pytest.mark.parametrize("nseq", [1, 2, 3, 65, 1000])
def test_bad_tables_are_dealt_inside(host, nseq):
    rng = np.random.default_rng(nseq)
    for i in range(12):
        T, groups, kvh = int(rng.integers(1, 300)), 32, int(rng.integers(1, 4))
        cu = ints(bad(rng, nseq, T))
        lens = ints(rng.choice([INT_MIN, -1, 0, 1, 239, 240, 241, INT_MAX], nseq))
        window, sinks = ((0, 0), (30, 4))[i % 2]
        for y in pieces(host, cu, lens, T, 16, 15, kvh, 1 + i % 3, 16, 64, window, sinks, 1, groups, 256):
            inside(y, nseq, T, kvh, groups)


@pytest.mark.parametrize("nseq", [512, 1024, 4096])
@pytest.mark.parametrize("kvh", [1, 3, 5])
def test_overlapping_requests_are_dealt_inside(host, nseq, kvh):
    """Every second request has all tokens behind 2^24 keys: the line is longer than f64 counts exactly, and cuts
    fall on the borders between threads."""
    rng = np.random.default_rng(nseq + kvh)
    T, groups = 65536 - int(rng.integers(0, 50)), 512
    cu = ints(np.where(np.arange(nseq + 1) % 2 == 0, 0, T))
    lens = ints(np.full(nseq, (1 << 24) - int(rng.integers(0, 100000))))
    for y in pieces(host, cu, lens, T, 16, 1 << 20, kvh, 256 // kvh, 16, 64, 0, 0, 1, groups, 256, most=2):
        inside(y, nseq, T, kvh, groups)
