"""Page tables that the GPU keeps: pages assigned and released, against loops over sequences and columns (whole numbers: equal)."""

import numpy as np
import pytest

from oracle import paged as op
from tests import _paged as P
from triton_llm import gpu
from triton_llm.kernels import assign_kv_pages, release_kv_pages

pytestmark = pytest.mark.gpu


def pool(rng, lens, page, max_pages, spare):
    """(table, free_pages, pages on the free list): every sequence's pages anywhere in the pool."""
    held = [min(max_pages, -(-max(int(n), 0) // page)) for n in lens]
    n_pages = max(1, sum(held) + spare)
    table = P.shuffled_table(rng, [h * page for h in held], page, max_pages, n_pages)
    rest = np.setdiff1d(np.arange(n_pages), table)
    free = np.full(n_pages, -7, np.int32)
    free[:rest.size] = rng.permutation(rest)
    return table, free, rest.size


def run_assign(lens, new, table, free, counts, page, tokens, in_place=False):
    lens_d, new_d, table_d, free_d, counts_d = map(P.int32, (lens, new, table, free, counts))
    out = tuple(P.int32(np.full(n, 99)) for n in (tokens, tokens, len(lens) + 1, len(lens)))
    counts_out = None if in_place else P.int32([5, 5])
    assign_kv_pages(lens_d, new_d, table_d, free_d, counts_d, page, tokens, out=out, counts_out=counts_out)
    got = [gpu.to_host(x) for x in (table_d, *out, counts_d if in_place else counts_out)]
    for name, g, w in zip(("table", "slots", "positions", "starts", "ends", "counts"), got,
                          op.assign(lens, new, table, free, counts, page, tokens)):
        np.testing.assert_array_equal(g, w, err_msg=name)
    for name, x, w in (("lens", lens_d, lens), ("new", new_d, new), ("free", free_d, free)):
        np.testing.assert_array_equal(gpu.to_host(x), w, err_msg=name)
    return got


@pytest.mark.parametrize("batch,page,hi,new_hi,spare,room", [
    (1, 16, 0, 1, 1, 0), (1, 16, 100, 40, 3, 5), (7, 16, 70, 3, 4, 0), (64, 32, 500, 1, 64, 0),
    (65, 16, 300, 200, 2000, 7), (300, 64, 1000, 90, 20, 0), (1024, 16, 64, 4, 2000, 3),
    (1025, 16, 64, 4, 700, 3),          # more sequences than one workgroup holds
    (2500, 16, 40, 9, 100000, 0),       # more rows too
    (5000, 16, 20, 3, 5000, 1),         # more than are searched in LDS
    (3, 1024, 5000, 9000, 30, 100), (20, 16, 200, 2000, 1500, 64)])
@pytest.mark.parametrize("in_place", [False, True])
def test_assign(batch, page, hi, new_hi, spare, room, in_place):
    rng = np.random.default_rng(batch + page)
    lens = rng.integers(0, hi, batch, endpoint=True)
    new = rng.integers(-1, new_hi, batch, endpoint=True)  # some rest
    lens[rng.integers(batch)] = hi // page * page
    max_pages = -(-(hi + new_hi) // page) + 1
    table, free, n = pool(rng, lens, page, max_pages, spare)
    run_assign(lens, new, table, free, [n, 3], page, int(np.maximum(new, 0).sum()) + room, in_place)


def test_assign_refuses_sequences_not_calls():
    """Too long for the table, a negative length, too many rows, too few pages: the others are granted."""
    rng = np.random.default_rng(1)
    page, max_pages = 16, 6
    lens = np.array([90, -3, 16, 5, 96, 0, 15, 32, 0, 2 ** 31 - 1, -2 ** 31])
    new = np.array([7, 2, 16, 0, 1, 40, 1, 33, 3, 2 ** 31 - 1, 2 ** 31 - 1])
    table, free, n = pool(rng, np.clip(lens, 0, 96), page, max_pages, 4)
    for count in (n, 0, 1, 2, -5, 1 << 30, free.size):
        for tokens in (120, 60, 17, 1, 0):
            run_assign(lens, new, table, free, [count, 0], page, tokens)
    free[:n] = [-1, free.size, 2 ** 31 - 1, 2][:n]  # a free list that names no pages
    run_assign(lens, new, table, free, [n, 0], page, 120)


def test_assign_without_rows_or_new_tokens():
    lens, new = np.array([3, 16, 0]), np.array([0, -4, 0])
    table, free, n = pool(np.random.default_rng(2), lens, 16, 3, 2)
    run_assign(lens, new, table, free, [n, 0], 16, 0)
    run_assign(lens, new, table, free, [n, 0], 16, 9000)


@pytest.mark.parametrize("batch,page,hi,spare", [(1, 16, 100, 3), (8, 16, 400, 0), (64, 32, 5000, 40), (512, 16, 16000, 9),
                                                 (1500, 16, 90, 5), (3, 1024, 300000, 2), (16, 16, 40000, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_release(batch, page, hi, spare, in_place):
    rng = np.random.default_rng(batch)
    lens = rng.integers(-2, hi, batch, endpoint=True)
    max_pages = max(1, -(-hi // page) - 1)  # some lengths pass the table
    table, free, n = pool(rng, lens, page, max_pages, spare)
    holes = rng.random(table.shape) < 0.05
    table[holes] = rng.choice([-1, free.size, 2 ** 31 - 1, -2 ** 31], int(holes.sum()))
    ended = rng.integers(0, 2, batch) * rng.choice([1, -1, 7], batch)
    for keep in (None, rng.integers(-1, max_pages + 2, batch)):
        lens_d, free_d, counts_d, table_d = P.int32(lens), P.int32(free), P.int32([n, 8]), P.int32(table)
        outs = {} if in_place else {"lens_out": P.int32(lens * 0 + 9), "counts_out": P.int32([1, 1])}
        left, counts = release_kv_pages(table_d, lens_d, P.int32(ended), free_d, counts_d, page,
                                        keep=None if keep is None else P.int32(keep), **outs)
        if not in_place:
            np.testing.assert_array_equal(gpu.to_host(lens_d), lens)
            np.testing.assert_array_equal(gpu.to_host(counts_d), [n, 8])
        w_free, w_counts, w_lens = op.release(table, lens, ended, free, [n, 8], page, keep)
        np.testing.assert_array_equal(gpu.to_host(free_d), w_free)
        np.testing.assert_array_equal(gpu.to_host(counts), w_counts)
        np.testing.assert_array_equal(gpu.to_host(left), w_lens)
        np.testing.assert_array_equal(gpu.to_host(table_d), table)


@pytest.mark.parametrize("batch", [4, 1100])
def test_release_past_the_stack(batch):
    """Pages given back twice: what has no room on the list is counted and dropped."""
    rng = np.random.default_rng(3)
    lens = np.full(batch, 32)
    table, free, n = pool(rng, lens, 16, 2, 3)
    free[:] = np.arange(free.size)
    for count in (free.size, free.size - 3, -1, 1 << 30):
        free_d, counts_d = P.int32(free), P.int32([count, 0])
        release_kv_pages(P.int32(table), P.int32(lens), P.int32(np.ones(batch)), free_d, counts_d, 16)
        w_free, w_counts, _ = op.release(table, lens, np.ones(batch), free, [count, 0], 16)
        np.testing.assert_array_equal(gpu.to_host(free_d), w_free)
        np.testing.assert_array_equal(gpu.to_host(counts_d), w_counts)


def test_many_steps_lose_no_page():
    """Sequences come, grow and end: every page is on the list or in one row, and a captured step replays with the lengths
    that are there then."""
    rng = np.random.default_rng(4)
    batch, page, max_pages, n_pages, tokens = 24, 16, 8, 120, 100
    lens = gpu.zeros((batch,), np.int32)
    table, free = P.int32(np.full((batch, max_pages), -1)), P.int32(rng.permutation(n_pages))
    counts, new, ended = P.int32([n_pages, 0]), gpu.zeros((batch,), np.int32), gpu.zeros((batch,), np.int32)
    out = tuple(gpu.zeros((n,), np.int32) for n in (tokens, tokens, batch + 1, batch))

    def step():
        release_kv_pages(table, lens, ended, free, counts, page)
        assign_kv_pages(lens, new, table, free, counts, page, tokens, out=out)
        gpu.copy_(lens, out[3])

    step()
    with gpu.capture() as graph:
        step()
    h_table, h_free, h_counts = gpu.to_host(table), gpu.to_host(free), gpu.to_host(counts)
    h_lens = np.zeros(batch, np.int64)
    for turn in range(40):
        h_end = (rng.random(batch) < 0.15).astype(np.int32)
        h_new = rng.integers(0, 9, batch).astype(np.int32)
        ended.from_numpy(h_end), new.from_numpy(h_new)
        graph.replay() if turn % 3 else step()
        h_free, h_counts, h_lens = op.release(h_table, h_lens, h_end, h_free, h_counts, page)
        h_table, slots, positions, starts, h_lens, h_counts = op.assign(h_lens, h_new, h_table, h_free, h_counts, page, tokens)
        for got, want in zip((table, free, counts, lens, *out), (h_table, h_free, h_counts, h_lens, slots, positions, starts, h_lens)):
            np.testing.assert_array_equal(gpu.to_host(got), want)
        used = [h_table[b, c] for b in range(batch) for c in range(-(-int(h_lens[b]) // page))]
        assert sorted(used + h_free[:h_counts[0]].tolist()) == list(range(n_pages))
