"""The page bookkeeping (qff.pages.PageTable) on the CPU: random sequences of
reservations, forks, releases and compactions against a model that keeps every
sequence's contents, the pools simulated with the copies the table asks for."""
import random

import numpy as np
import pytest

from qff.pages import OutOfPages, PageTable


class Pool:
    """Pages of position values, copied as the table asks."""

    def __init__(self, t, pages):
        self.t, self.data = t, np.zeros((pages, t.page_size), np.int64)

    def copy(self, pairs):
        assert len({d for _, d in pairs}) == len(pairs) and not {s for s, _ in pairs} & {d for _, d in pairs}
        for s, d in pairs:
            self.data[d] = self.data[s]

    def write(self, slot, start, values):
        for i, v in enumerate(values, start):
            page = self.t._rows[slot, i // self.t.page_size]
            assert self.t.refs[page] == 1
            self.data[page, i % self.t.page_size] = v

    def read(self, slot):
        n, ps = self.t.lengths[slot], self.t.page_size
        return [int(self.data[self.t._rows[slot, i // ps], i % ps]) for i in range(n)]


def _consistent(t):
    held = np.bincount(np.concatenate([np.array(t.pages_of(s), np.int64) for s in range(len(t.lengths))]), minlength=len(t.refs))
    assert np.array_equal(held, t.refs)
    assert sorted(t._free) == [p for p in range(len(t.refs)) if not held[p]]


@pytest.mark.parametrize("seed", range(12))
def test_random_operations(seed):
    rng = random.Random(seed)
    ps, slots = 16, 7
    t = PageTable(60, ps, slots, 30 * ps, device="cpu")
    pool, model, value = Pool(t, 60), [[] for _ in range(slots)], 0
    for _ in range(400):
        s, op = rng.randrange(slots), rng.random()
        if op < 0.6:
            start = len(model[s]) if rng.random() < 0.85 else rng.randrange(len(model[s]) + 1)
            end = min(start + rng.choice([1, 1, 2, ps, 3 * ps + 1]), 30 * ps)
            if start >= end:
                continue
            rows, free = t._rows.copy(), t.free_pages
            try:
                pool.copy(t.reserve(s, start, end))
            except OutOfPages:
                assert np.array_equal(rows, t._rows) and free == t.free_pages
                continue
            new = list(range(value, value + end - start))
            value += end - start
            pool.write(s, start, new)
            model[s][start:end] = new
        elif op < 0.8:
            d = rng.randrange(slots)
            if d == s or model[d]:
                with pytest.raises(ValueError):
                    t.fork(s, d)
            else:
                t.fork(s, d)
                model[d] = list(model[s])
        elif op < 0.93:
            t.release(s)
            model[s] = []
        else:
            src, dst = t.compact()
            pool.copy(list(zip(src, dst)))
            used = int((t.refs > 0).sum())
            assert (t.refs[:used] > 0).all()
        _consistent(t)
        for k in range(slots):
            assert t.lengths[k] == len(model[k]) and pool.read(k) == model[k]
        t.sync()
        assert np.array_equal(t.table.numpy(), t._rows)
        # whatever is grouped is held by all of the group, and nothing before a slot's length is missing
        g, sh = t.group.numpy(), t.shared_len.numpy()
        for k in range(1, slots):
            if g[k] >= 0 and g[k] == g[k - 1]:
                first = int(np.flatnonzero(g == g[k])[0])
                m = min(sh[g == g[k]])
                assert 64 <= m <= min(t.lengths[k], t.lengths[first])
                assert model[k][:m] == model[first][:m]


def test_copy_on_write_keeps_what_others_hold():
    t = PageTable(10, 16, 3, 64, device="cpu")
    assert t.reserve(0, 0, 20) == []
    t.fork(0, 1)
    t.fork(0, 2)
    assert t.free_pages == 8 and t.pages_of(1) == [0, 1]
    assert t.reserve(1, 20, 21) == [(1, 2)]     # position 20 goes to the shared second page
    assert t.reserve(0, 20, 21) == [(1, 3)]
    assert t.reserve(2, 20, 21) == []           # the last holder keeps it
    assert [t.pages_of(s) for s in range(3)] == [[0, 3], [0, 2], [0, 1]]
    # a page rewritten whole is not copied
    t.release(0)
    t.fork(1, 0)
    assert t.reserve(0, 0, 32) == []
    assert t.lengths[0] == 32 and set(t.pages_of(0)).isdisjoint(t.pages_of(1))


def test_groups():
    t = PageTable(100, 16, 8, 1024, device="cpu")
    t.reserve(0, 0, 200)
    for d in (1, 2):
        t.fork(0, d)
        t.reserve(d, 200, 201)
    t.reserve(4, 0, 80)
    t.fork(4, 5)
    t.fork(4, 6)
    t.reserve(6, 64, 65)
    t.reserve(7, 0, 30)
    g, s = t.groups()
    # 0-2: 200 positions less the last page, which 0 still shares with nobody; 4 and 5 share all 80, 6 the 64 before its own page
    assert g.tolist() == [0, 0, 0, -1, 4, 4, 4, -1]
    assert s.tolist() == [192, 192, 192, 0, 64, 80, 64, 0]
    t.release(1)
    assert t.groups()[0].tolist() == [-1, -1, -1, -1, 4, 4, 4, -1]


def test_groups_split_where_less_than_half_is_shared():
    t = PageTable(100, 16, 4, 1024, device="cpu")
    t.reserve(0, 0, 640)
    t.fork(0, 1)
    t.fork(0, 2)
    t.reserve(2, 100, 640)     # shares 96 positions with 0 and 1, which share 640
    t.fork(2, 3)
    g, s = t.groups()
    assert g.tolist() == [0, 0, 2, 2] and s.tolist() == [640, 640, 640, 640]


def test_refusals():
    for args in ((0, 16, 1, 64), (1, 16, 0, 64), (1, 16, 1, 0), (1, 8, 1, 64), (1, 48, 1, 64), (1, 8192, 1, 64)):
        with pytest.raises(ValueError):
            PageTable(*args, device="cpu")
    t = PageTable(4, 16, 2, 64, device="cpu")
    for start, end in ((1, 2), (0, 0), (-1, 1), (0, 65)):
        with pytest.raises(ValueError):
            t.reserve(0, start, end)
    t.reserve(0, 0, 64)
    with pytest.raises(OutOfPages):
        t.reserve(1, 0, 1)
    with pytest.raises(ValueError):
        t.fork(0, 0)
    assert t.compact() == ([], [])


def test_truncate_is_what_reserving_less_leaves():
    t = PageTable(10, 16, 3, 128, device="cpu")
    t.reserve(0, 0, 50)
    t.fork(0, 1)
    for slot, end in ((0, 51), (0, -1), (2, 1)):
        with pytest.raises(ValueError):
            t.truncate(slot, end)
    t.truncate(0, 50)                       # all of it: nothing changes
    assert t.pages_of(0) == [0, 1, 2, 3]
    t.truncate(0, 32)                       # pages 2 and 3 are slot 1's alone
    assert t.pages_of(0) == [0, 1] and t.lengths == [32, 50, 0] and t.free_pages == 6
    assert t.refs[:4].tolist() == [2, 2, 1, 1]
    t.truncate(1, 33)
    assert t.pages_of(1) == [0, 1, 2] and t.free_pages == 7
    t.sync()
    assert t.table.tolist() == t._rows.tolist() and t.group.tolist() == [-1, -1, -1] and t._rows[1, 3] == -1
    t.truncate(1, 0)
    assert t.pages_of(1) == [] and t.refs[:3].tolist() == [1, 1, 0]
    assert t.reserve(1, 0, 16) == [] and t.lengths == [32, 16, 0]
    _consistent(t)
