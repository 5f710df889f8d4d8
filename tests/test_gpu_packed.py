"""Packed batches on the GPU: appends by slots (bits as the padded append's) and attention of packed rows."""

import numpy as np
import pytest

from oracle import numerics as on
from oracle import paged as op
from tests import _paged as P
from triton_llm import gpu
from triton_llm.kernels import (paged_attention_packed, paged_attention_prefill, paged_kv_append_slots,
                                precompute_cos_sin)

pytestmark = pytest.mark.gpu
DTYPES = ["float32", "float16", "bfloat16"]


@pytest.mark.parametrize("dtype,Hq,Hkv,D,page,n,rotary,inter,in_place", [
    ("bfloat16", 24, 8, 128, 16, 1, 128, False, True),
    ("float16", 15, 5, 64, 32, 333, 32, True, False),
    ("float32", 9, 3, 64, 16, 100, 64, False, False),
    ("bfloat16", 4, 2, 128, 64, 77, 64, False, True),
    ("bfloat16", 4, 4, 64, 16, 3, 0, False, False),
    ("float16", 2, 1, 6, 16, 40, 4, False, False),   # rows of no round size
    ("bfloat16", 2, 1, 10, 16, 40, 6, True, True),
    ("float32", 2, 2, 24, 128, 130, 12, False, True),
    ("float16", 2, 1, 16, 1024, 7, 2, True, False),
])
@pytest.mark.parametrize("with_q", [True, False])
def test_append_slots(dtype, Hq, Hkv, D, page, n, rotary, inter, in_place, with_q):
    rng = np.random.default_rng(n)
    n_pages = n // page + 5
    slots = rng.permutation(n_pages * page)[:n].astype(np.int32)
    rows = 60
    positions = rng.integers(0, rows, n).astype(np.int32)
    if n > 3:
        slots[1], slots[2] = -1, n_pages * page
        slots[n // 2] = -2 ** 31
        positions[n - 1], positions[n - 2] = rows, -1  # outside the angles
    shape = (n_pages, Hkv, page, D)
    kp, vp = P.values(rng, shape, dtype), P.values(rng, shape, dtype)
    q, k, v = (P.values(rng, (n, h, D), dtype) for h in (Hq, Hkv, Hkv))
    before = P.values(rng, q.shape, dtype)
    cos, sin = precompute_cos_sin(rows, rotary) if rotary else (None, None)
    tab = [gpu.to_device(x) if x is not None else None for x in (cos, sin)]
    q_d, kp_d, vp_d = P.dev(q, dtype) if with_q else None, P.dev(kp, dtype), P.dev(vp, dtype)
    qo_d = None if in_place or not with_q else P.dev(before, dtype)
    out = paged_kv_append_slots(q_d, P.dev(k, dtype), P.dev(v, dtype), kp_d, vp_d, P.int32(slots),
                                P.int32(positions) if rotary else None, *tab, q_out=qo_d, interleaved=inter)
    # a token of a batch of its own, whose table names its page and whose position is its slot's place there
    wq, wk, wv = (q if in_place else before).copy(), kp.copy(), vp.copy()
    for t in range(n):
        if not 0 <= slots[t] < n_pages * page or (rotary and not 0 <= positions[t] < rows):
            continue
        one = [np.repeat(x[positions[t]][None], page, 0) if x is not None else None for x in (cos, sin)]
        qt, wk, wv = op.append(q[None, t:t + 1], k[None, t:t + 1], v[None, t:t + 1], wk, wv,
                               np.array([[slots[t] // page]]), np.array([slots[t] % page]), *one, interleaved=inter, dtype=dtype)
        wq[t] = qt[0, 0]
    bits = {2: np.uint16, 4: np.uint32}[kp.dtype.itemsize]
    pairs = [("k", kp_d, wk), ("v", vp_d, wv)] + ([("q", out, wq)] if with_q else [])
    assert with_q or out is None
    for name, got, exp in pairs:
        np.testing.assert_array_equal(gpu.to_host(got).view(bits), exp.view(bits), err_msg=name)


def run_packed(dtype, Hq, Hkv, D, page, lens, new, window, sinks, behind=3, max_new=None, counts=False, seed=0):
    rng = np.random.default_rng(seed)
    lens, new = np.asarray(lens, np.int32), np.asarray(new, np.int32)
    max_new = int(new.max()) if max_new is None else max_new
    total = lens + new
    max_pages = max(1, -(-int(total.max()) // page))
    n_pages = sum(-(-max(int(t), 0) // page) for t in total) + 2
    table = P.shuffled_table(rng, total, page, max_pages, n_pages)
    keep = [np.arange(max_pages * page) < t for t in total]
    kp, vp = (P.pool_with(rng, table, keep, (n_pages, Hkv, page, D), dtype) for _ in range(2))
    starts = np.concatenate([[0], np.cumsum(new)]) + behind  # rows of no sequence before and behind
    rows = int(starts[-1]) + behind
    q, before = P.values(rng, (rows, Hq, D), dtype), P.values(rng, (rows, Hq, D), dtype)
    out = P.dev(before, dtype)
    paged_attention_packed(P.dev(q, dtype), P.dev(kp, dtype), P.dev(vp, dtype), P.int32(table), P.int32(lens), P.int32(starts),
                           Hq, Hkv, max_new, window=window, sinks=sinks, out=out, host_new_lens=new.tolist() if counts else None)
    got, old = P.back(out, dtype), on.from_storage(before, dtype)
    kf, vf = on.from_storage(kp, dtype), on.from_storage(vp, dtype)
    untouched = np.ones(rows, bool)
    for b, (n, m) in enumerate(zip(lens, np.minimum(new, max_new))):
        if m == 0:
            continue
        at = slice(starts[b], starts[b] + m)
        untouched[at] = False
        k, there = op.gather(kf, table[b], max(int(total[b]), 1))
        v, _ = op.gather(vf, table[b], max(int(total[b]), 1))
        want, tol = P.rows_want(q[at].transpose(1, 0, 2), k, v, n + np.arange(m), there, window, sinks, D ** -0.5, dtype)
        P.check(f"packed {dtype} {Hq}/{Hkv} d{D} window {window} sequence {b}", got[at].transpose(1, 0, 2), want, tol)
    np.testing.assert_array_equal(got[untouched], old[untouched])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,page,window,sinks", [(64, 16, 0, 0), (128, 32, 0, 0), (64, 16, 40, 3), (128, 128, 100, 0),
                                                 (64, 1024, 130, 70)])
@pytest.mark.parametrize("counts", [False, True])
def test_packed(dtype, D, page, window, sinks, counts):
    run_packed(dtype, 4, 2, D, page, [0, 1, 333, 5, 64, -3, 700], [150, 129, 37, 0, 1, 20, 1], window, sinks, counts=counts)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (5, 1), (9, 3), (12, 12), (40, 1)])
def test_packed_groups_and_single_tokens(Hq, Hkv):
    run_packed("bfloat16", Hq, Hkv, 64, 16, [0, 99, 3, 1000, 0, 17], [1] * 6, 0, 0)
    run_packed("float32", Hq, Hkv, 64, 16, [0, 99, 3, 1000, 0, 17], [1, 1, 30, 1, 2, 1], 0, 0)
    run_packed("float16", Hq, Hkv, 128, 32, [0, 99, 3, 1000, -2, 17, 500], [1, 1, 30, 2, 3, 1, 6], 70, 20)
    run_packed("float32", Hq, Hkv, 128, 64, [0, 99, 3, 1000, -2, 17, 500], [1, 1, 3, 2, 3, 1, 6], 1, 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_packed_few_rows_every_length(dtype, D):
    """Row tiles of up to 32 rows: blocks, rings and page look-ups that end everywhere; divided keys and whole ones."""
    lens = [0, 14, 15, 16, 31, 48, 63, 64, 65, 127, 129, 191, 255, 300, 1100]
    run_packed(dtype, 4, 2, D, 16, lens, [1] * len(lens), 0, 0)
    run_packed(dtype, 8, 1, D, 16, lens, [1, 2, 3, 4] * 3 + [4, 1, 2], 0, 0)
    run_packed(dtype, 3, 1, D, 64, [9000, 5], [1, 2], 0, 0)
    run_packed(dtype, 3, 1, D, 16, [9000, 5], [5, 1], 3000, 100)


def test_packed_pages_that_are_not_there():
    rng = np.random.default_rng(9)
    Hq, Hkv, D, page = 4, 2, 64, 16
    lens, new = np.array([60, 200, 30], np.int32), np.array([1, 3, 40], np.int32)
    total = lens + new
    for dtype in DTYPES:
        table = P.shuffled_table(rng, total, page, 14, 40)
        table[0, 1], table[1, 5], table[1, 12], table[2, 0], table[2, 3] = -1, 40, 2 ** 31 - 1, -5, -1
        keep = [np.arange(14 * page) < t for t in total]
        kp, vp = (P.pool_with(rng, table, keep, (40, Hkv, page, D), dtype) for _ in range(2))
        starts = np.concatenate([[0], np.cumsum(new)])
        q = P.values(rng, (int(starts[-1]), Hq, D), dtype)
        got = P.back(paged_attention_packed(P.dev(q, dtype), P.dev(kp, dtype), P.dev(vp, dtype), P.int32(table), P.int32(lens),
                                            P.int32(starts), Hq, Hkv, 40), dtype)
        for b in range(3):
            at = slice(starts[b], starts[b + 1])
            k, there = op.gather(on.from_storage(kp, dtype), table[b], int(total[b]))
            v, _ = op.gather(on.from_storage(vp, dtype), table[b], int(total[b]))
            want, tol = P.rows_want(q[at].transpose(1, 0, 2), k, v, lens[b] + np.arange(new[b]), there, 0, 0, D ** -0.5, dtype)
            P.check(f"packed without pages {dtype} sequence {b}", got[at].transpose(1, 0, 2), want, tol)


def test_packed_many_sequences():
    rng = np.random.default_rng(6)
    new = rng.integers(0, 4, 150)
    new[77] = 200
    run_packed("float16", 4, 2, 64, 16, rng.integers(0, 90, 150), new, 0, 0)


def test_packed_rows_past_max_new_stay():
    run_packed("bfloat16", 3, 1, 64, 16, [10, 20, 30], [40, 70, 5], 0, 0, max_new=40)


def test_packed_starts_outside_the_rows():
    """Starts past the rows or before them: only rows that there are count."""
    rng = np.random.default_rng(7)
    Hq, Hkv, D, page, rows = 2, 1, 64, 16, 30
    q, before = P.values(rng, (rows, Hq, D), "bfloat16"), P.values(rng, (rows, Hq, D), "bfloat16")
    kp, vp = P.values(rng, (9, Hkv, page, D), "bfloat16"), P.values(rng, (9, Hkv, page, D), "bfloat16")
    table = np.array([[0, 1, 2], [3, 4, 5], [6, 7, 8]], np.int32)
    out = P.dev(before, "bfloat16")
    paged_attention_packed(P.dev(q, "bfloat16"), P.dev(kp, "bfloat16"), P.dev(vp, "bfloat16"), P.int32(table), P.int32([0, 9, 0]),
                           P.int32([-5, 20, 44, 2 ** 31 - 1]), Hq, Hkv, 30, out=out)
    got = P.back(out, "bfloat16")
    kf, vf = on.from_storage(kp, "bfloat16"), on.from_storage(vp, "bfloat16")
    for b, lo, hi, n in ((0, 0, 20, 0), (1, 20, 30, 9)):
        k, there = op.gather(kf, table[b], n + hi - lo)
        v, _ = op.gather(vf, table[b], n + hi - lo)
        want, tol = P.rows_want(q[lo:hi].transpose(1, 0, 2), k, v, n + np.arange(hi - lo), there, 0, 0, D ** -0.5, "bfloat16")
        P.check(f"packed starts sequence {b}", got[lo:hi].transpose(1, 0, 2), want, tol)


def test_packed_starts_that_go_back():
    """A start far below the one before it: the sequence before has no rows, and none are read or written for it."""
    rng = np.random.default_rng(17)
    Hq, Hkv, D, page, rows = 2, 1, 64, 16, 30
    q, before = P.values(rng, (rows, Hq, D), "float32"), P.values(rng, (rows, Hq, D), "float32")
    kp, vp = P.values(rng, (9, Hkv, page, D), "float32"), P.values(rng, (9, Hkv, page, D), "float32")
    table = np.array([[0, 1, 2], [3, 4, 5]], np.int32)
    out = P.dev(before, "float32")
    paged_attention_packed(P.dev(q, "float32"), P.dev(kp, "float32"), P.dev(vp, "float32"), P.int32(table), P.int32([0, 9]),
                           P.int32([7, -2 ** 31, 11]), Hq, Hkv, 30, out=out)
    got = P.back(out, "float32")
    k, there = op.gather(on.from_storage(kp, "float32"), table[1], 20)
    v, _ = op.gather(on.from_storage(vp, "float32"), table[1], 20)
    want, tol = P.rows_want(q[:11].transpose(1, 0, 2), k, v, 9 + np.arange(11), there, 0, 0, D ** -0.5, "float32")
    P.check("packed starts that go back", got[:11].transpose(1, 0, 2), want, tol)
    np.testing.assert_array_equal(got[11:], before[11:])


def test_append_slots_of_more_rows_than_the_caches():
    """40 MB of rows in one call, bit for bit what calls of a third of them leave."""
    rng = np.random.default_rng(18)
    Hq, Hkv, D, page, n, rows = 24, 8, 128, 64, 3900, 500
    n_pages = -(-n // page) + 2
    q, k, v = (P.values(rng, (n, h, D), "bfloat16") for h in (Hq, Hkv, Hkv))
    slots = rng.permutation(n_pages * page)[:n].astype(np.int32)
    positions = rng.integers(0, rows, n).astype(np.int32)
    tab = [gpu.to_device(x) for x in precompute_cos_sin(rows, D)]
    shape = (n_pages, Hkv, page, D)
    got = []
    for pieces in (1, 3):
        kp, vp = (P.dev(np.zeros(shape, np.uint16), "bfloat16") for _ in range(2))
        outs = []
        for at in np.array_split(np.arange(n), pieces):
            outs.append(gpu.to_host(paged_kv_append_slots(*(P.dev(x[at], "bfloat16") for x in (q, k, v)), kp, vp, P.int32(slots[at]),
                                                          P.int32(positions[at]), *tab)))
        got.append((np.concatenate(outs), gpu.to_host(kp), gpu.to_host(vp)))
    for a, b in zip(*got):
        np.testing.assert_array_equal(a.view(np.uint16), b.view(np.uint16))


@pytest.mark.parametrize("dtype,D", [("bfloat16", 128), ("float32", 64)])
def test_packed_is_padded(dtype, D):
    """The same rows padded: equal where both divide the keys alike, which sequences of one length do not change."""
    rng = np.random.default_rng(8)
    Hq, Hkv, page, n, B = 6, 2, 16, 40, 3
    lens = np.array([100, 0, 260], np.int32)
    table = P.shuffled_table(rng, lens + n, page, 20, 60)
    kp, vp = (P.values(rng, (60, Hkv, page, D), dtype) for _ in range(2))
    q = P.values(rng, (B, n, Hq, D), dtype)
    args = P.dev(kp, dtype), P.dev(vp, dtype), P.int32(table), P.int32(lens)
    want = P.back(paged_attention_prefill(P.dev(q, dtype), *args, Hq, Hkv), dtype)
    got = P.back(paged_attention_packed(P.dev(q.reshape(B * n, Hq, D), dtype), *args, P.int32(np.arange(B + 1) * n), Hq, Hkv, n),
                 dtype)
    weight = np.abs(on.from_storage(vp, dtype)).max()
    # both are within half a step of the rounded weights and of the output of the same value
    assert np.abs(got - want.reshape(got.shape)).max() <= 2 * (2 * P.HALF_STEP[dtype] + 400 * 2.0 ** -24) * weight * 1.1
