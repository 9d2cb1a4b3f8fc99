"""The index arithmetic that ragged calls do on the device (attention_shared.hip:
seq_of, own_span; linear_scan.hip: span_of, first_unit, unit_seq, entry), replayed
on the host, where a wrong index is an assertion: over tables that fit, every row
and unit is found once, and over tables that do not, every index that is read or
written stays inside its buffer.
"""
import numpy as np
import pytest

INT_MIN, INT_MAX = -2 ** 31, 2 ** 31 - 1


def wrap(x):
    """x as 32-bit arithmetic leaves it."""
    return (x - INT_MIN) % 2 ** 32 + INT_MIN


class Table:
    """A device table: reads outside it fail."""

    def __init__(self, values):
        self.values = [int(x) for x in values]

    def __getitem__(self, i):
        assert 0 <= i < len(self.values), f"read of entry {i} of {len(self.values)}"
        return self.values[i]


def fitting(rng, nseq, T):
    """Offsets from 0, some sequences empty, up to a few rows behind the last one."""
    total = int(rng.integers(0, T + 1))
    return np.concatenate([[0], np.sort(rng.integers(0, total + 1, nseq - 1)), [total]])


def bad(rng, nseq, T):
    kind = rng.integers(0, 4)
    if kind == 0:
        return rng.integers(INT_MIN, INT_MAX, nseq + 1, endpoint=True)
    if kind == 1:
        return rng.integers(-T, 2 * T + 1, nseq + 1)
    table = fitting(rng, nseq, T)
    if kind == 2:  # a fitting one with a few entries replaced
        at = rng.integers(0, nseq + 1, 3)
        table[at] = rng.choice([INT_MIN, -1, 0, T, T + 1, INT_MAX], 3)
        return table
    return table[::-1].copy()


# ---------------------------------------------------------------------------- shared-prefix attention
def seq_of(cu, nseq, t):
    lo, width = 0, nseq
    while width > 0:
        step = (width + 63) // 64
        n = 0
        for lane in range(64):
            i = lane * step + step - 1
            n += i < width and cu[lo + i + 1] <= t
        lo += n * step
        width = min(step - 1, width - n * step)
    return lo if lo < nseq and cu[lo] <= t else -1


def own_span(cu, start, length, T, max_keys, nkeys, s, t):
    first = min(max(start[s], 0), nkeys)
    n = min(max(length[s], 0), min(max_keys, nkeys - first))
    left = max(wrap(min(cu[s + 1], T) - 1 - t), 0)
    return first, max(n - left, 0)


@pytest.mark.parametrize("nseq", [1, 2, 63, 64, 65, 130, 4096])
def test_rows_find_their_sequence(nseq):
    rng = np.random.default_rng(nseq)
    for _ in range(3):
        T = int(rng.integers(1, 3 * nseq + 2))
        values = fitting(rng, nseq, T)
        cu = Table(values)
        for t in rng.integers(0, T, 40):
            t = int(t)
            want = int(np.searchsorted(values[1:], t, side="right"))
            assert seq_of(cu, nseq, t) == (want if want < nseq else -1)


@pytest.mark.parametrize("nseq", [1, 2, 3, 64, 65, 200, 4096])
def test_bad_attention_tables_stay_inside(nseq):
    rng = np.random.default_rng(nseq)
    for _ in range(12):
        T, nkeys = int(rng.integers(1, 65537)), int(rng.integers(1, 1 << 20))
        max_keys = int(rng.integers(1, 2 * nkeys))
        cu = Table(bad(rng, nseq, T))
        start = Table(rng.choice([INT_MIN, -1, 0, 1, nkeys - 1, nkeys, nkeys + 1, INT_MAX], nseq))
        length = Table(rng.choice([INT_MIN, -1, 0, 1, 7, nkeys, INT_MAX], nseq))
        for t in rng.integers(0, T, 25):
            s = seq_of(cu, nseq, int(t))
            assert -1 <= s < nseq
            if s >= 0:
                first, count = own_span(cu, start, length, T, max_keys, nkeys, s, int(t))
                assert 0 <= first <= nkeys and 0 <= count <= max_keys and first + count <= nkeys


# ---------------------------------------------------------------------------- linear scan
class Units:
    """The unit numbering of one call, as every work-group computes it."""

    def __init__(self, values, nseq, T, unit):
        self.cu, self.nseq, self.T, self.unit = Table(values), nseq, T, unit
        self.nunits = T // unit + nseq
        self.entries = T // unit

    def clamp(self, x):
        return min(max(x, 0), self.T)

    def span(self, s):
        t0 = self.clamp(self.cu[s])
        return t0, min(max(self.cu[s + 1], t0), self.T)

    def first(self, s):
        return self.clamp(self.cu[s]) // self.unit + s

    def seq(self, u):
        lo, width = 0, self.nseq
        while width > 1:
            step = (width + 63) // 64
            found = [lane for lane in range(64) if lane * step < width and self.first(lo + lane * step) <= u]
            n = found[-1] if found else 0
            lo += n * step
            width = min(step, width - n * step)
        return lo

    def entry(self, s, i):
        at = self.clamp(self.cu[s]) // self.unit + i - 1
        assert 0 <= at < self.entries, f"entry {at} of {self.entries}"
        return at

    def walk(self):
        """(sequence, unit of it, first token, token behind the last) of the work-groups that do not leave at
        once, their entries checked."""
        for u in range(self.nunits):
            s = self.seq(u)
            t0, t1 = self.span(s)
            index = u - self.first(s)
            begin = t0 + index * self.unit
            assert INT_MIN <= begin <= INT_MAX and INT_MIN <= begin + self.unit <= INT_MAX
            end = min(begin + self.unit, t1)
            if index < 0 or (index > 0 and begin >= t1):
                continue
            assert 0 <= begin <= end <= self.T
            if end != t1:
                self.entry(s, index + 1)  # what the unit adds
            if index > 0:
                self.entry(s, index)      # what it starts from
            yield s, index, begin, end

    def join(self):
        used = []
        for s in range(self.nseq):
            t0, t1 = self.span(s)
            used += [self.entry(s, i) for i in range(1, (t1 - t0 + self.unit - 1) // self.unit)]
        return used


CALLS = [(1, 700, 64), (3, 700, 128), (64, 5000, 64), (65, 4096, 128), (200, 300, 64), (1000, 5000, 320),
         (7, 1 << 20, 1 << 14)]


@pytest.mark.parametrize("nseq,T,unit", CALLS)
def test_units_cover_each_sequence_once(nseq, T, unit):
    rng = np.random.default_rng(nseq)
    for _ in range(3):
        values = fitting(rng, nseq, T)
        units = Units(values, nseq, T, unit)
        got = list(units.walk())
        want = [(s, i, a + i * unit, min(a + (i + 1) * unit, b)) for s, (a, b) in enumerate(zip(values, values[1:]))
                for i in range(max(1, -(-(b - a) // unit)))]
        assert sorted(got) == sorted((s, i, int(a), int(b)) for s, i, a, b in want)
        used = units.join()
        assert len(used) == len(set(used))


@pytest.mark.parametrize("nseq,T,unit", CALLS + [(4096, 1 << 20, 1 << 20), (4096, 4096, 64)])
def test_bad_unit_tables_stay_inside(nseq, T, unit):
    rng = np.random.default_rng(nseq + T)
    for _ in range(2 if nseq == 4096 else 12):
        units = Units(bad(rng, nseq, T), nseq, T, unit)
        for _ in units.walk():
            pass
        units.join()


def test_missing_starts_and_lengths_are_refused():
    torch = pytest.importorskip("torch")
    clef = pytest.importorskip("clef_hip")
    q, gate = torch.zeros(4, 2, 64), torch.zeros(2, 4, 64)
    k, vt = torch.zeros(2, 16, 64), torch.zeros(2, 64, 16)
    cu, table = torch.tensor([0, 1, 2], dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for starts, lens in ((None, table), (table, None), (None, None)):
        with pytest.raises(clef.ClefError, match="int32 device tensor"):
            clef.attention_gated_shared(q, k, vt, gate, cu, starts, lens)
