"""Attention that reads a shared prefix once, against the 64-bit form of plain paged attention.  Positions that a call may not
read hold NaN; tolerances are those derived in tests/_paged.py."""

import ctypes

import numpy as np
import pytest

from oracle import numerics as on
from oracle import paged as op
from tests import _paged as P
from triton_llm import gpu
from triton_llm.kernels import (allocate_kv_pages, paged_attention_decode, paged_attention_shared, plan_shared_attention,
                                shared_workspace_bytes)

pytestmark = pytest.mark.gpu
DTYPES = ["float32", "float16", "bfloat16"]


class Case:
    """Sequences of lens tokens; groups: [(members, shared positions)].  A group's shared positions lie in its first
    member's pages; the other members' tables name them too, or nothing at all (whole shared pages are not looked up there)."""

    def __init__(self, dtype, Hq, Hkv, D, page, lens, groups, seed=0, blind=True, edit=None):
        rng = np.random.default_rng(seed)
        self.dtype, self.heads, self.page, self.groups = dtype, (Hq, Hkv, D), page, groups
        self.lens = lens = np.asarray(lens, np.int64)
        B, max_pages = len(lens), max(1, -(-int(max(lens.max(), 1)) // page))
        n_pages = sum(-(-max(int(n), 0) // page) for n in lens) + 2
        self.table = P.shuffled_table(rng, lens, page, max_pages, n_pages)
        for members, shared in groups:
            first = next((m for m in members if 0 <= m < B and lens[m] >= shared), None)
            for m in members:
                if first is not None and 0 <= m < B and lens[m] >= shared and m != first:
                    n = -(-shared // page)
                    self.table[m, :n] = self.table[first, :n]
        if edit:
            edit(self.table, n_pages)
        keep = [np.arange(max_pages * page) < n for n in lens]
        shape = (n_pages, Hkv, page, D)
        self.kp, self.vp = (P.pool_with(rng, self.table, keep, shape, dtype) for _ in range(2))
        self.q = P.values(rng, (B, Hq, D), dtype)
        self.device_table = self.table.copy()
        if blind:  # only the first sequence's entries are read for whole shared pages
            for members, shared in groups:
                inside = [m for m in members if 0 <= m < B and lens[m] >= shared]
                for m in inside[1:]:
                    self.device_table[m, :shared // page] = -1

    def lists(self):
        members = [m for g, _ in self.groups for m in g]
        members += [-1] * (len(self.lens) - len(members))
        starts = np.concatenate([[0], np.cumsum([len(g) for g, _ in self.groups])])
        return members, starts, [s for _, s in self.groups]

    def run(self, len_add=0, scale=None, name="shared"):
        Hq, Hkv, D = self.heads
        scale = D ** -0.5 if scale is None else scale
        members, starts, shared = self.lists()
        before = P.values(np.random.default_rng(99), self.q.shape, self.dtype)
        out, table = P.dev(before, self.dtype), P.int32(self.device_table)
        plan = plan_shared_attention(table, P.int32(self.lens - len_add), P.int32(members), P.int32(starts), P.int32(shared), Hq,
                                     Hkv, D, self.page, P.H.GPU_DTYPES[self.dtype], len_add=len_add)
        paged_attention_shared(P.dev(self.q, self.dtype), P.dev(self.kp, self.dtype), P.dev(self.vp, self.dtype), table, plan, Hq,
                               Hkv, sm_scale=scale, out=out)
        got = P.back(out, self.dtype)
        listed = sorted({m for m in members if 0 <= m < len(self.lens)})
        rest = np.setdiff1d(np.arange(len(self.lens)), listed)
        np.testing.assert_array_equal(got[rest], on.from_storage(before, self.dtype)[rest])
        clean = [np.where(np.isnan(on.from_storage(x, self.dtype)), 0, x).astype(x.dtype) for x in (self.kp, self.vp)]
        want, tol = P.decode_want(self.q, *clean, self.table, self.lens, 0, 0, scale, self.dtype)
        if self.dtype != "float32":
            # weights of many rows are rounded to the type; of few rows they are in two words, the second of which is
            most = max([len(g) for g, n in self.groups if n > 0] + [1]) * (Hq // Hkv)
            rounding = P.HALF_STEP[self.dtype] ** (1 if most > 32 else 2)
            kf, vf = (on.from_storage(x, self.dtype) for x in clean)
            for b in listed:
                n = int(min(max(self.lens[b], 0), self.table.shape[1] * self.page))
                if n == 0:
                    continue
                k, there = op.gather(kf, self.table[b], n)
                v, _ = op.gather(vf, self.table[b], n)
                for h in range(Hq):
                    _, w = op.attend(on.from_storage(self.q[b, h:h + 1], self.dtype), k[h // (Hq // Hkv)], v[h // (Hq // Hkv)],
                                     there[None], scale)
                    tol[b, h] += rounding * w[0] * 1.05
        P.check(f"{name} {self.dtype} {Hq}/{Hkv} d{D} page {self.page}", got[listed], want[listed], tol[listed])
        return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page,shared", [(16, 16), (16, 160), (32, 96), (256, 256), (1024, 1024), (16, 0), (16, 37), (64, 65),
                                         (32, 31), (16, 1)])
def test_lengths(dtype, D, page, shared):
    """Own parts of every length round a block and a tile, none among them; shared parts of whole pages and of any length."""
    own = [0, 1, 15, 16, 17, 31, 33, 63, 64, 65, 200]
    Case(dtype, 6, 2, D, page, [shared + n for n in own], [(list(range(len(own))), shared)]).run()


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (4, 2), (4, 1), (5, 1), (14, 2), (9, 9), (40, 1), (128, 1)])
@pytest.mark.parametrize("dtype,D", [("bfloat16", 128), ("float32", 64), ("float16", 64), ("float32", 128)])
def test_heads(Hq, Hkv, dtype, D):
    Case(dtype, Hq, Hkv, D, 16, [150, 100, 96, 230], [([2, 0, 3, 1], 96)]).run()


@pytest.mark.parametrize("dtype", DTYPES)
def test_groups(dtype):
    """Groups of several sizes and none, in any order; sequences alone, short of the shared part, empty, in no group."""
    lens = [300, 90, 0, 301, 64, 500, 95, 420, 1, 96, 700, 33]
    groups = [([5, 0, 3], 256), ([], 64), ([10], 300), ([1, 9, 4, 6], 64), ([7], 0), ([2, 8], 16), ([99], 5)]
    Case(dtype, 6, 2, 64, 16, lens, groups).run()


@pytest.mark.parametrize("dtype", DTYPES)
def test_shorter_than_the_shared_part(dtype):
    """Members with fewer tokens than the group shares read their own pages; one that is left shares nothing."""
    Case(dtype, 4, 2, 64, 16, [200, 50, 0, 230, 128], [([1, 0, 2, 3, 4], 128)]).run()
    Case(dtype, 4, 2, 64, 16, [200, 50, 0, 20], [([1, 0, 2, 3], 128)]).run()


@pytest.mark.parametrize("dtype,D,batch", [("bfloat16", 128, 70), ("float16", 64, 130), ("float32", 64, 70)])
def test_many_rows(dtype, D, batch):
    """Several tiles of rows over one prefix, rows of a sequence in two of them."""
    rng = np.random.default_rng(2)
    Case(dtype, 6, 2, D, 16, 700 + rng.integers(0, 60, batch), [(rng.permutation(batch).tolist(), 699)]).run()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("batch,group,page,shared", [(11, 3, 16, 401), (16, 3, 16, 33), (16, 4, 64, 1000), (21, 3, 32, 95), (13, 5, 16, 64),
                                                     (63, 3, 16, 130)])
def test_up_to_64_rows(dtype, D, batch, group, page, shared):
    """33 to 64 rows in a tile, over few keys and many; tiles with a page that is not there, in their first half and their second."""
    rng = np.random.default_rng(25)

    def edit(table, n_pages):
        if shared > 90 and page == 16:
            table[:, 1], table[:, 6] = -1, n_pages
    Case(dtype, group, 1, D, page, shared + rng.integers(0, 40, batch), [(rng.permutation(batch).tolist(), shared)], edit=edit).run()


def test_more_sequences_than_a_workgroup_plans_at_once():
    rng = np.random.default_rng(3)
    B = 1100
    members = rng.permutation(B)
    lens = np.zeros(B, np.int64)
    groups = []
    for i, at in enumerate(np.array_split(members, 400)):
        shared = int(rng.integers(0, 60))
        lens[at] = shared + rng.integers(0, 30, at.size)
        groups.append((at.tolist(), shared))
    Case("bfloat16", 2, 1, 64, 16, lens, groups).run()


@pytest.mark.parametrize("dtype", DTYPES)
def test_long(dtype):
    Case(dtype, 3, 1, 128, 64, [9000, 5100, 8200, 5000], [([0, 1, 2, 3], 4992)]).run()
    Case(dtype, 3, 1, 64, 16, [9000, 3000], [([0, 1], 16)]).run()


def test_fewer_compute_units(monkeypatch):
    for cus in (1, 3, 40):
        P.H.set_override(monkeypatch, "TRITON_LLM_HIP_MAX_CUS", cus)
        Case("bfloat16", 6, 2, 64, 16, [700, 0, 1300, 515, 1000], [([0, 2, 3, 4, 1], 512)]).run()
        Case("float32", 6, 2, 64, 16, [700, 0, 1300, 515, 1000], [([0, 2, 3, 4, 1], 512)]).run()


def test_scales_and_len_add():
    for scale in (-0.2, 0.0, 4.0):
        Case("float16", 2, 1, 64, 16, [90, 70, 65], [([0, 1, 2], 64)]).run(scale=scale)
    Case("bfloat16", 2, 1, 64, 16, [90, 70, 65], [([0, 1, 2], 64)]).run(len_add=1)
    Case("bfloat16", 2, 1, 64, 16, [90, 70, 65], [([0, 1, 2], 64)]).run(len_add=-7)


@pytest.mark.parametrize("dtype", DTYPES)
def test_pages_that_are_not_there(dtype):
    def edit(table, n_pages):
        table[:, 1] = -1            # hidden in the shared part
        table[0, 5], table[1, 6], table[2, 4] = n_pages, 2 ** 31 - 1, -2 ** 31
    Case(dtype, 3, 1, 64, 16, [100, 130, 70, 64], [([0, 1, 2, 3], 64)], edit=edit).run()

    def none(table, n_pages):
        table[:, :] = -1
    got = Case(dtype, 3, 1, 64, 16, [100, 130, 70, 64], [([0, 1, 2, 3], 64)], edit=none).run()
    assert (got == 0).all()


def test_lengths_past_the_table():
    c = Case("bfloat16", 2, 1, 64, 16, [96, 96, 50], [([0, 1, 2], 32)])
    c.lens = np.array([1 << 30, 2 ** 31 - 1, 50])
    c.run()


def test_a_sequence_named_twice():
    """It counts where it is named last."""
    c = Case("bfloat16", 4, 2, 64, 16, [96, 130, 50, 70], [([0, 3, 1, 1], 32)])
    c.run()
    c = Case("bfloat16", 4, 2, 64, 16, [96, 130, 50, 200], [([0, 1, 3], 64), ([3], 16)], blind=False)
    c.run()


def test_starts_that_go_back():
    """Groups that overlap by their starts: nobody shares, and every sequence is right."""
    c = Case("float16", 4, 2, 64, 16, [96, 130, 70, 50], [([0, 1, 2, 3], 32)], blind=False)
    c.lists = lambda: ([0, 1, 2, 3], [0, 4, 0, 4], [32, 32, 32])
    c.run()
    c.lists = lambda: ([0, 1, 2, 3], [-3, 2, 77], [32, -5])
    c.run()
    # in all no more than there are sequences, and some of them in two groups
    c = Case("float16", 4, 2, 64, 16, [96, 130, 70, 50, 64, 33, 90, 41], [(list(range(8)), 32)], blind=False)
    c.lists = lambda: (list(range(8)), [0, 4, 2, 6, 8], [32, 16, 32, 16])
    c.run()


@pytest.mark.parametrize("batch,n_groups", [(6, 1500), (1, 1), (300, 2), (130, 3), (500, 40), (513, 2), (1030, 1)])
def test_more_groups_than_a_workgroup_plans_at_once(batch, n_groups):
    """Groups without members among those with some; a thread a group, and more groups or sequences than threads."""
    rng = np.random.default_rng(23)
    members = rng.permutation(batch)
    cuts = np.sort(rng.integers(0, batch + 1, n_groups - 1))
    groups = [(at.tolist(), 40) for at in np.split(members, cuts)]
    Case("float16", 2, 1, 64, 16, 40 + rng.integers(0, 20, batch), groups).run()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,Hq,Hkv,batch,shared", [(64, 6, 2, 130, 48), (128, 20, 10, 60, 37), (64, 28, 7, 90, 16), (128, 40, 2, 150, 0), (64, 3, 3, 1100, 21),
                                                   (64, 66, 2, 140, 16)])
def test_many_short_sequences(dtype, D, Hq, Hkv, batch, shared):
    """Own parts of one tile and fewer, of two now and then, in such numbers that they fill the device."""
    rng = np.random.default_rng(26)
    lens = shared + rng.integers(0, 17, batch)
    lens[::9] += rng.integers(14, 60, lens[::9].size)
    def edit(table, n_pages):
        table[3::7, -1] = -1
    Case(dtype, Hq, Hkv, D, 16, lens, [(rng.permutation(batch).tolist(), shared)], edit=edit).run()


@pytest.mark.parametrize("batch", [5, 1100])
def test_lengths_below_zero(batch):
    """Sequences of no positions, as a padded batch's: zeros, and no part in what the others share."""
    rng = np.random.default_rng(24)
    lens = np.where(np.arange(batch) % 3 == 1, -7, 50 + rng.integers(0, 9, batch))
    got = Case("bfloat16", 2, 1, 64, 16, lens, [(list(range(batch)), 48)]).run()
    assert not got[lens < 0].any()


def test_a_prefix_beyond_32_bit_offsets():
    """A 5 GiB pool: shared and own pages at its end."""
    rng = np.random.default_rng(9)
    dtype, Hq, Hkv, D, page = "bfloat16", 2, 1, 128, 1024
    n_pages = 5 * (1 << 30) // (page * D * 2)
    kp, vp = allocate_kv_pages(n_pages, Hkv, page, D, P.H.GPU_DTYPES[dtype], zero=False)
    k, v = P.values(rng, (1, Hkv, page, D), dtype), P.values(rng, (1, Hkv, page, D), dtype)

    def place(pool, at, x):
        t = gpu.DeviceTensor(ctypes.c_void_p(pool.data_ptr() + at * x.nbytes), x.shape, pool.dtype, x.nbytes, defer_free=False)
        gpu.copy_(t, P.dev(x, dtype))
        gpu.synchronize()

    for at in (n_pages - 1, n_pages - 2):
        place(kp, at, k), place(vp, at, v)
    lens = [1024 + 70, 1024 + 3]
    table = np.array([[n_pages - 1, n_pages - 2], [-1, n_pages - 2]], np.int32)
    q = P.values(rng, (2, Hq, D), dtype)
    plan = plan_shared_attention(P.int32(table), P.int32(lens), P.int32([0, 1]), P.int32([0, 2]), P.int32([1024]), Hq, Hkv, D, page,
                                 P.H.GPU_DTYPES[dtype])
    got = P.back(paged_attention_shared(P.dev(q, dtype), kp, vp, P.int32(table), plan, Hq, Hkv), dtype)
    kf, vf = (np.concatenate([on.from_storage(x, dtype)[0]] * 2, 1) for x in (k, v))
    for b, n in enumerate(lens):
        want, tol = P.rows_want(q[b][:, None], kf[:, :n], vf[:, :n], [n - 1], np.ones(n, bool), 0, 0, D ** -0.5, dtype)
        P.check(f"far pages sequence {b}", got[b][:, None], want, tol)


def test_a_plan_serves_every_layer_and_a_captured_step():
    """Two layers by one plan; captured, and replayed with other lengths, tables and groups."""
    rng = np.random.default_rng(11)
    dtype, Hq, Hkv, D, page, B, max_pages = "bfloat16", 6, 2, 64, 16, 5, 12
    n_pages = B * max_pages
    pools = [tuple(P.values(rng, (n_pages, Hkv, page, D), dtype) for _ in "kv") for _ in range(2)]
    dev_pools = [tuple(P.dev(x, dtype) for x in kv) for kv in pools]
    q = [P.values(rng, (B, Hq, D), dtype) for _ in range(2)]
    q_d, out = [P.dev(x, dtype) for x in q], [gpu.zeros((B, Hq, D), P.H.GPU_DTYPES[dtype]) for _ in q]
    table, lens, members = gpu.zeros((B, max_pages), np.int32), gpu.zeros((B,), np.int32), gpu.zeros((B,), np.int32)
    starts, shared = gpu.zeros((4,), np.int32), gpu.zeros((3,), np.int32)
    ws = gpu.allocate((shared_workspace_bytes(B, 3, Hq, Hkv, D),), np.uint8)
    state = {"plan": None}

    def step():
        state["plan"] = plan_shared_attention(table, lens, members, starts, shared, Hq, Hkv, D, page, P.H.GPU_DTYPES[dtype],
                                              plan=state["plan"])
        for x, (kp, vp), o in zip(q_d, dev_pools, out):
            paged_attention_shared(x, kp, vp, table, state["plan"], Hq, Hkv, out=o, workspace=ws)

    step()
    with gpu.capture() as graph:
        step()
    for turn in range(6):
        h_table = rng.permutation(n_pages).reshape(B, max_pages).astype(np.int32)
        h_members, n = rng.permutation(B).astype(np.int32), int(rng.integers(2, B + 1))
        h_starts = np.array([0, n, n, B], np.int32)
        h_shared = rng.integers(0, 100, 3).astype(np.int32)
        for g in range(3):
            at = h_members[h_starts[g]:h_starts[g + 1]]
            h_table[at, :-(-h_shared[g] // page)] = h_table[at[:1], :-(-h_shared[g] // page)]
        h_lens = rng.integers(100, max_pages * page, B).astype(np.int32)
        for t, h in ((table, h_table), (lens, h_lens), (members, h_members), (starts, h_starts), (shared, h_shared)):
            t.from_numpy(h)
        graph.replay()
        for i in range(2):
            got = P.back(out[i], dtype)
            want, tol = P.decode_want(q[i], *pools[i], h_table, h_lens, 0, 0, D ** -0.5, dtype)
            tol = tol + P.HALF_STEP[dtype] * np.abs(on.from_storage(pools[i][1], dtype)).max() * 1.05
            P.check(f"replay {turn} layer {i}", got, want, tol)
        replayed = [gpu.to_host(o) for o in out]
        step()  # eager, between replays
        for o, r in zip(out, replayed):
            np.testing.assert_array_equal(gpu.to_host(o), r)


def test_a_plan_of_other_sizes_is_not_followed():
    """At the C entry, where nothing else keeps a plan and its sizes together: the output stays."""
    c = Case("bfloat16", 4, 2, 64, 16, [96, 130, 50], [([0, 1, 2], 32)])
    members, starts, shared = c.lists()
    plan = plan_shared_attention(P.int32(c.table), P.int32(c.lens), P.int32(members), P.int32(starts), P.int32(shared), 4, 2, 64, 16,
                                 P.H.GPU_DTYPES["bfloat16"])
    plan.sizes = plan.sizes[:1] + (plan.sizes[1] + 1,) + plan.sizes[2:]  # a wider table than it was made for
    wide = np.pad(c.table, ((0, 0), (0, 1)), constant_values=-1)
    before = P.values(np.random.default_rng(0), c.q.shape, "bfloat16")
    out = P.dev(before, "bfloat16")
    paged_attention_shared(P.dev(c.q, "bfloat16"), P.dev(c.kp, "bfloat16"), P.dev(c.vp, "bfloat16"), P.int32(wide), plan, 4, 2, out=out)
    np.testing.assert_array_equal(P.back(out, "bfloat16"), on.from_storage(before, "bfloat16"))


@pytest.mark.parametrize("dtype", DTYPES)
def test_as_decode_and_deterministic(dtype):
    """Beside paged_attention_decode over the same pages, and equal when it is run again."""
    c = Case(dtype, 6, 2, 128, 16, [300, 290, 257, 411], [([3, 1, 0, 2], 256)], blind=False)
    Hq, Hkv, D = c.heads
    a, b = c.run(), c.run()
    np.testing.assert_array_equal(a, b)
    plain = P.back(paged_attention_decode(P.dev(c.q, dtype), P.dev(c.kp, dtype), P.dev(c.vp, dtype), P.int32(c.table),
                                          P.int32(c.lens), Hq, Hkv), dtype)
    finite = on.from_storage(c.vp, dtype)
    weight = np.abs(finite[np.isfinite(finite)]).max()
    assert np.abs(a - plain).max() <= (3 * P.HALF_STEP[dtype] + 1000 * 2.0 ** -24) * weight
