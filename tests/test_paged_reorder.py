"""Reordering beams touches the pages in which a slot and its parent differ, not those that they share."""

import numpy as np

from triton_llm.paged_cache import PageTables


class Counted(PageTables):
    drops = 0

    def _drop(self, page):
        self.drops += 1
        super()._drop(page)


def beams(n_items, J, tokens, page=16):
    t = Counted(n_items * (tokens // page + 2 + 2 * J), page, n_items * J, tokens + 64)
    for i in range(n_items):
        for _ in range(J):
            t.open()
    t.begin([tokens if s % J == 0 else 0 for s in range(n_items * J)])
    t.advance()
    t.reorder([s for s in range(n_items * J) if s % J], [s // J * J for s in range(n_items * J) if s % J])
    t.begin([1] * (n_items * J))
    t.advance()
    t.take_edits()
    return t


def test_a_step_costs_what_changes():
    n_items, J, tokens = 4, 8, 2003
    t = beams(n_items, J, tokens)
    rng = np.random.default_rng(0)
    for _ in range(20):
        slots = list(range(n_items * J))
        parents = [s // J * J + int(rng.integers(J)) for s in slots]
        before = [list(x) for x in t.tables]
        refs = list(t.refs)
        t.drops = 0
        t.reorder(slots, parents)
        changed = sum(a != b for s, p in zip(slots, parents) for a, b in zip(before[s], before[p]))
        assert t.tables == [before[p] for p in parents]
        assert t.drops <= changed <= 3 * n_items * J  # of about 126 pages a slot
        _, edits = t.take_edits()
        assert len(edits) == changed
        count = [0] * t.n_pages
        for pages in t.tables:
            for p in pages:
                count[p] += 1
        assert count == t.refs and sorted(t._free) == [p for p in range(t.n_pages) if not count[p]]
        assert sum(refs) == sum(t.refs)
        t.begin([1] * (n_items * J))
        t.advance()
        t.take_edits()


def test_parents_of_other_lengths():
    t = PageTables(40, 16, 4, 200)
    for _ in range(4):
        t.open()
    t.begin([100, 20, 0, 37])
    t.advance()
    t.reorder([0, 1, 2, 3], [1, 0, 0, 2])
    assert t.lens == [20, 100, 100, 0] and [len(x) for x in t.tables] == [2, 7, 7, 0]
    assert t.tables[1] == t.tables[2] and t.tables[1] is not t.tables[2]
    assert t.free_pages == 40 - 2 - 7 and [t.refs[p] for p in t.tables[1]] == [2] * 7
    t.reorder([1, 2], [3, 3])
    assert t.free_pages == 38
