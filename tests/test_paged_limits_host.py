"""A cache that its steps could not use is refused when it is made, not by the first step."""

import pytest

from triton_llm.paged_cache import PagedKVCache, PageTables

GOOD = {"n_pages": 4, "page_size": 16, "max_batch": 2, "max_seq": 32}


@pytest.mark.parametrize("change,msg", [
    ({"page_size": 0}, "power of 2"), ({"page_size": -16}, "power of 2"), ({"page_size": 24}, "power of 2"),
    ({"page_size": 2048}, "power of 2"), ({"window": 1 << 31}, "window and sinks"), ({"sinks": 1 << 31}, "window and sinks"),
    ({"max_seq": (1 << 30) + 1}, "max_seq"), ({"max_batch": 65536}, "max_batch")])
def test_refused_when_made(change, msg):
    with pytest.raises(ValueError, match=msg):
        PagedKVCache(1, 4, 2, 64, **{**GOOD, **change})


@pytest.mark.parametrize("page_size", [0, -16])
def test_tables_alone_refuse(page_size):
    with pytest.raises(ValueError, match="page_size must be positive"):
        PageTables(**{**GOOD, "page_size": page_size})


def test_more_blocks_than_attention_counts():
    for heads, change in [((4, 4), {"max_batch": 64, "max_seq": 1 << 27}), ((64, 2), {"max_batch": 64, "max_seq": 1 << 26}),
                          ((2, 2), {"max_batch": 1024, "max_seq": 1 << 28, "window": 1 << 25})]:
        with pytest.raises(ValueError, match="2\\^31"):
            PagedKVCache(1, *heads, 64, **{**GOOD, **change})


def test_largest_are_taken():
    assert PageTables(n_pages=4, page_size=10, max_batch=1, max_seq=95).max_pages == 10  # on the host any size
    t = PageTables(n_pages=4, page_size=1024, max_batch=1, max_seq=1 << 30, window=(1 << 31) - 1, sinks=(1 << 31) - 1)
    assert t.max_pages == 1 << 20
