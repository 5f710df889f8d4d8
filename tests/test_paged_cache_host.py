"""The page tables of the paged cache on the host: who has which pages, what a step needs, refusals."""

import numpy as np
import pytest

from triton_llm.paged_cache import PagedKVCache, PageTables


class Mirror:
    """What the GPU would hold: pages of tokens and a table that follow the edits, checked against every sequence."""

    def __init__(self, t):
        self.t = t
        self.pages = np.full((t.n_pages, t.page_size), -1, np.int64)
        self.table = np.full((t.max_batch, t.max_pages), -1)
        self.seqs = {}
        self.stamp = 0

    def publish(self):
        copies, edits = self.t.take_edits()
        for a, b in copies:
            self.pages[b] = self.pages[a]
        for (s, c), p in edits.items():
            self.table[s, c] = p

    def step(self, new):
        self.t.begin(new)
        self.publish()
        for s, n in enumerate(new):
            for _ in range(n):
                at = len(self.seqs[s])
                self.stamp += 1
                self.pages[self.table[s, at // self.t.page_size], at % self.t.page_size] = self.stamp
                self.seqs[s].append(self.stamp)
        self.t.advance()

    def check(self):
        self.publish()
        t, ps = self.t, self.t.page_size
        count = np.zeros(t.n_pages, int)
        for s in range(t.max_batch):
            pages = t.tables[s]
            assert (pages is not None) == (s in self.seqs)
            row = [] if pages is None else pages
            assert self.table[s, :len(row)].tolist() == row and (self.table[s, len(row):] == -1).all()
            for p in row:
                if p >= 0:
                    count[p] += 1
            if pages is None:
                continue
            toks = self.seqs[s]
            assert t.lens[s] == len(toks)
            for at, tok in enumerate(toks):
                visible = not t.window or at > len(toks) - t.window or at < t.sinks
                if visible:  # to the next token
                    assert self.pages[row[at // ps], at % ps] == tok
        assert count.tolist() == t.refs
        assert sorted(t._free) == [p for p in range(t.n_pages) if count[p] == 0]


@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3), (16, 0), (1, 17), (50, 16)])
def test_random_use(window, sinks):
    rng = np.random.default_rng(window + sinks)
    t = PageTables(60, 16, 6, 200, window, sinks)
    m = Mirror(t)
    for _ in range(400):
        slots = sorted(m.seqs)
        act = rng.integers(0, 7)
        if act == 0 and len(slots) < 6:
            m.seqs[t.open()] = []
        elif act == 1 and slots and len(slots) < 6:
            a = int(rng.choice(slots))
            m.seqs[t.fork(a)] = list(m.seqs[a])
        elif act == 2 and len(slots) > 1 and rng.random() < 0.5:
            a = int(rng.choice(slots))
            t.close(a)
            del m.seqs[a]
        elif act == 3 and len(slots) > 1:
            some = [int(s) for s in rng.permutation(slots)[:rng.integers(1, len(slots) + 1)]]
            parents = [int(rng.choice(slots)) for _ in some]
            t.reorder(some, parents)
            taken = [list(m.seqs[p]) for p in parents]
            for s, x in zip(some, taken):
                m.seqs[s] = x
        elif act == 4:
            t.compact()
            used = sum(r > 0 for r in t.refs)
            assert all(t.refs[:used]) and not any(t.refs[used:])
        elif slots:
            new = [0] * 6
            for s in slots:
                new[s] = min(int(rng.choice([0, 1, 1, 1, 5, 40])), 200 - len(m.seqs[s]))
            before = (list(t.refs), [list(x) if x is not None else None for x in t.tables], list(t.lens))
            if any(new):
                try:
                    m.step(new)
                except ValueError as e:
                    assert "pages needed" in str(e)
                    assert before == (list(t.refs), [list(x) if x is not None else None for x in t.tables], list(t.lens))
                    a = slots[0]
                    t.close(a)
                    del m.seqs[a]
        m.check()


def test_forks_share_full_pages_and_copy_the_last():
    t = PageTables(10, 16, 4, 100)
    a = t.open()
    t.begin([20, 0, 0, 0])
    t.advance()
    b, c = t.fork(a), t.fork(a)
    assert t.free_pages == 8 and t.refs[t.tables[a][0]] == 3
    t.begin([1, 1, 1, 0])
    copies, _ = t.take_edits()
    assert len(copies) == 2 and t.free_pages == 6  # the last of the three keeps the page
    assert t.tables[a][0] == t.tables[b][0] == t.tables[c][0] and len({x[1] for x in (t.tables[a], t.tables[b], t.tables[c])}) == 3


def test_refusals_change_nothing():
    t = PageTables(3, 16, 2, 40)
    with pytest.raises(ValueError, match="slot 0 is not open"):
        t.begin([1, 0])
    a = t.open()
    for new, msg in [([41, 0], "exceeds max_seq"), ([1], "entry for each"), ([0, 0], "at least one"), ([-1, 0], ">= 0"),
                     ([1, 1], "slot 1 is not open")]:
        with pytest.raises(ValueError, match=msg):
            t.begin(new)
    with pytest.raises(ValueError, match="no step has begun"):
        t.advance()
    t.begin([30, 0])
    for call in (lambda: t.begin([1, 0]), lambda: t.open(), lambda: t.close(a), lambda: t.fork(a), lambda: t.compact(),
                 lambda: t.reorder([a], [a])):
        with pytest.raises(ValueError, match="a step has begun"):
            call()
    t.advance()
    b = t.fork(a)
    with pytest.raises(ValueError, match="all 2 slots"):
        t.open()
    with pytest.raises(ValueError, match="3 pages needed, 1 free"):
        t.begin([10, 10])  # a page each, and a copy of the shared last one
    assert t.free_pages == 1 and t.lens == [30, 30]
    for slots, parents, msg in [([a], [a, b], "1 slots, 2 parents"), ([a, a], [a, b], "twice"), ([a], [5], "not open"),
                                ([-1], [a], "not open")]:
        with pytest.raises(ValueError, match=msg):
            t.reorder(slots, parents)
    t.close(b)
    with pytest.raises(ValueError, match="not open"):
        t.close(b)


def test_window_gives_pages_back():
    t = PageTables(8, 16, 1, 1000, window=32, sinks=4)
    t.open()
    for _ in range(300):
        t.begin([1])
        t.advance()
        assert 8 - t.free_pages <= 4  # the sinks' page and a window's
    assert t.tables[0][0] >= 0 and t.tables[0][1] == -1


@pytest.mark.parametrize("args,kw,msg", [
    ((2, 10, 3, 64), {}, "bad head counts"), ((0, 9, 3, 64), {}, "bad head counts"),
    ((2, 9, 3, 96), {}, "d_k in"), ((2, 9, 3, 64), {"n_pages": 0}, "must be positive"), ((2, 9, 3, 64), {"max_seq": 0}, "must be positive"),
    ((2, 9, 3, 64), {"window": -1}, "window and sinks"), ((2, 9, 3, 64), {"page_size": 24}, "power of 2")])
def test_constructor_refuses(args, kw, msg):
    with pytest.raises(ValueError, match=msg):
        PagedKVCache(*args, **{"n_pages": 4, "max_batch": 2, "max_seq": 32, **kw})
