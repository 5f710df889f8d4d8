"""Refusals of the GPU's page tables, packed batches and shared-prefix attention: every call here is refused, or has nothing to
do, before any device work, in the Python layer and at the C entries; and their oracles against the host's page tables."""

import ctypes

import numpy as np
import pytest

from oracle import paged as op
from triton_llm import _lib, gpu
from triton_llm.kernels import (SharedPlan, assign_kv_pages, paged_attention_packed, paged_attention_shared,
                                paged_kv_append_slots, pages_workspace_bytes, plan_shared_attention, release_kv_pages,
                                shared_workspace_bytes)
from triton_llm.paged_cache import PagedKVCache, PageTables

F32, BF16, BAD = _lib.DTYPE_F32, _lib.DTYPE_BF16, 99


def fake(shape, dtype=np.float32):
    return gpu.DeviceTensor(ctypes.c_void_p(None), shape, dtype, 0, defer_free=False)


def i32(*shape):
    return fake(shape, np.int32)


POOL = (9, 2, 16, 64)


def call(fn, defaults, change):
    a = dict(defaults)
    a.update(change)
    kw = {n[1:]: a.pop(n) for n in list(a) if n.startswith("_")}
    return fn(*a.values(), **kw)


RELEASE = dict(table=i32(3, 7), lens=i32(3), ended=i32(3), free=i32(9), counts=i32(2), page=16)
ASSIGN = dict(lens=i32(3), new=i32(3), table=i32(3, 7), free=i32(9), counts=i32(2), page=16, tokens=5)


@pytest.mark.parametrize("change,msg", [
    ({"table": fake((3, 7))}, "page_table must be int32"), ({"table": i32(3)}, "page_table must be int32"),
    ({"table": i32(3, 0)}, "page_table must be int32"), ({"lens": i32(4)}, "lens must be int32 of shape"),
    ({"lens": fake((3,))}, "lens must be int32"), ({"free": i32(3, 3)}, "free_pages must be int32"),
    ({"free": i32(0)}, "free_pages must be int32"), ({"counts": i32(1)}, "counts must be int32 of shape"),
    ({"counts": fake((2,))}, "counts must be int32"), ({"page": 24}, "power of 2"), ({"page": 8}, "power of 2"),
    ({"free": i32(1 << 27)}, "exceed"), ({"table": i32(3, 1 << 27)}, "exceed"), ({"_counts_out": i32(3)}, "counts must be"),
])
def test_release_and_assign_refuse(change, msg):
    for fn, defaults in ((release_kv_pages, RELEASE), (assign_kv_pages, dict(ASSIGN, _out=(i32(5), i32(5), i32(4), i32(3))))):
        with pytest.raises(ValueError, match=msg):
            call(fn, defaults, change)


@pytest.mark.parametrize("change,msg", [({"ended": i32(2)}, "ended must be int32"), ({"_keep": i32(2)}, "keep must be int32"),
                                        ({"_keep": fake((3,))}, "keep must be int32"), ({"_lens_out": i32(4)}, "lens_out must")])
def test_release_refuses(change, msg):
    with pytest.raises(ValueError, match=msg):
        call(release_kv_pages, RELEASE, change)


@pytest.mark.parametrize("change,msg", [
    ({"new": i32(2)}, "new_lens must be int32"), ({"tokens": -1}, "max_tokens"), ({"tokens": 1 << 31}, "max_tokens"),
    ({"_out": (i32(5), i32(5), i32(4))}, "out must be"), ({"_out": (i32(4), i32(5), i32(4), i32(3))}, "slots must be"),
    ({"_out": (i32(5), i32(6), i32(4), i32(3))}, "positions must"), ({"_out": (i32(5), i32(5), i32(3), i32(3))}, "starts must"),
    ({"_out": (i32(5), i32(5), i32(4), fake((3,)))}, "ends must"),
])
def test_assign_refuses(change, msg):
    with pytest.raises(ValueError, match=msg):
        call(assign_kv_pages, dict(ASSIGN, _out=(i32(5), i32(5), i32(4), i32(3))), change)


def test_pages_batch_limit():
    assert pages_workspace_bytes(0) == pages_workspace_bytes(65536) == 0 and pages_workspace_bytes(65535) >= 4 * 65535
    with pytest.raises(ValueError, match="at most 65535"):
        release_kv_pages(i32(65536, 2), i32(65536), i32(65536), i32(9), i32(2), 16)


SLOTS = dict(q=fake((5, 4, 64)), k=fake((5, 2, 64)), v=fake((5, 2, 64)), kp=fake(POOL), vp=fake(POOL), slots=i32(5),
             positions=i32(5), cos=fake((50, 32)), sin=fake((50, 32)))


@pytest.mark.parametrize("change,msg", [
    ({"kp": fake((9, 2, 16))}, "matching 4-D"), ({"vp": fake((9, 2, 32, 64))}, "matching 4-D"),
    ({"kp": fake((1 << 27, 2, 16, 64)), "vp": fake((1 << 27, 2, 16, 64))}, "exceed"),
    ({"k": fake((5, 3, 64))}, "k_new shape"), ({"k": fake((1, 5, 2, 64))}, "k_new shape"), ({"v": fake((4, 2, 64))}, "v_new shape"),
    ({"slots": i32(4)}, "slots must be int32"), ({"slots": fake((5,))}, "slots must be int32"),
    ({"positions": i32(4)}, "positions must be int32"), ({"positions": fake((5,))}, "positions must be int32"),
    ({"positions": None}, "without positions"), ({"q": fake((4, 4, 64))}, "does not match k_new"),
    ({"q": fake((5, 3, 64))}, "multiple of n_kv_head"), ({"q": None, "_q_out": fake((5, 4, 64))}, "without q_dev"),
    ({"_q_out": fake((5, 2, 64))}, "out must be like q"), ({"v": fake((5, 2, 64), np.float16)}, "share one dtype"),
    ({"cos": None}, "both be given"), ({"cos": fake((50, 33)), "sin": fake((50, 33))}, "cos/sin tables"),
    ({"cos": fake((50, 32), np.float64), "sin": fake((50, 32), np.float64)}, "cos/sin tables"),
])
def test_append_slots_refuses(change, msg):
    with pytest.raises(ValueError, match=msg):
        call(paged_kv_append_slots, SLOTS, change)


PACKED = dict(q=fake((8, 4, 64)), kp=fake(POOL), vp=fake(POOL), table=i32(3, 7), lens=i32(3), starts=i32(4), n_head=4, n_kv_head=2,
              max_new=5, _out=fake((8, 4, 64)))


@pytest.mark.parametrize("change,msg", [
    ({"starts": i32(3)}, "starts must be int32"), ({"starts": fake((4,))}, "must be int32"), ({"lens": i32(2)}, "cache_lens"),
    ({"q": fake((8, 4, 32))}, "q shape"), ({"q": fake((2, 4, 4, 64))}, "q shape"), ({"n_kv_head": 4}, "KV heads"),
    ({"n_head": 5}, "multiple of n_kv_head"), ({"max_new": -1}, "max_new"), ({"_window": -1}, "window and sinks"),
    ({"_sinks": 1 << 31}, "window and sinks"), ({"vp": fake(POOL, np.float16)}, "share one dtype"),
    ({"_out": fake((7, 4, 64))}, "out must be like q"), ({"table": i32(3, 1 << 27)}, "exceed"),
    ({"_host_new_lens": [1, 2]}, "host_new_lens"), ({"kp": fake((9, 2, 16, 32)), "vp": fake((9, 2, 16, 32))}, "d_k in"),
])
def test_packed_refuses(change, msg):
    with pytest.raises(ValueError, match=msg):
        call(paged_attention_packed, PACKED, change)


def test_packed_without_rows():
    for change in ({"max_new": 0}, {"q": fake((0, 4, 64)), "_out": fake((0, 4, 64))}):
        a = dict(PACKED, **change)
        assert call(paged_attention_packed, a, {}) is a["_out"]


PLAN = dict(table=i32(3, 7), lens=i32(3), members=i32(3), starts=i32(3), shared=i32(2), n_head=4, n_kv_head=2, d_k=64, page=16,
            dtype=np.float32)


@pytest.mark.parametrize("change,msg", [
    ({"table": fake((3, 7))}, "page_table must be int32"), ({"table": i32(3, 0)}, "page_table"), ({"lens": i32(2)}, "cache_lens"),
    ({"members": i32(4)}, "members must be int32"), ({"members": fake((3,))}, "members must be int32"),
    ({"starts": i32(2)}, "shared_lens must be"), ({"shared": i32(0), "starts": i32(1)}, "shared_lens must be"),
    ({"shared": fake((2,))}, "shared_lens must be int32"), ({"n_head": 5}, "multiple of n_kv_head"), ({"d_k": 32}, "d_k in"),
    ({"page": 20}, "power of 2"), ({"table": i32(3, 1 << 27)}, "exceed"), ({"n_head": 129, "n_kv_head": 1}, "not supported"),
    ({"dtype": np.int32}, "unsupported dtype"),
])
def test_plan_refuses(change, msg):
    with pytest.raises(ValueError, match=msg):
        call(plan_shared_attention, PLAN, change)


def plan_of(*sizes):
    p = SharedPlan.__new__(SharedPlan)
    p.sizes, p.buffer = sizes, fake((64,), np.uint8)
    return p


SHARED = dict(q=fake((3, 4, 64)), kp=fake(POOL), vp=fake(POOL), table=i32(3, 7), plan=plan_of(3, 7, 2, 4, 2, 64, 16, F32), n_head=4,
              n_kv_head=2, _out=fake((3, 4, 64)))


@pytest.mark.parametrize("change,msg", [
    ({"q": fake((3, 4, 32))}, "q shape"), ({"q": fake((2, 4, 64))}, "q shape"), ({"table": fake((3, 7))}, "must be int32"),
    ({"n_kv_head": 4}, "KV heads"), ({"vp": fake(POOL, np.float16)}, "share one dtype"), ({"_out": fake((3, 4, 32))}, "like q"),
    ({"table": i32(3, 8)}, "the plan is for"), ({"plan": plan_of(3, 7, 2, 8, 2, 64, 16, F32)}, "the plan is for"),
    ({"plan": plan_of(3, 7, 2, 4, 2, 64, 16, BF16)}, "dtype code"),
])
def test_shared_refuses(change, msg):
    with pytest.raises(ValueError, match=msg):
        call(paged_attention_shared, SHARED, change)


# ---- the C entries ---------------------------------------------------------------------

NULL, PTR = ctypes.c_void_p(None), ctypes.c_void_p(0x100000)  # PTR is never followed: the calls are refused


def at(i):
    """An address of its own for each argument, 1 MiB apart."""
    return ctypes.c_void_p(0x10000000 + (i << 20))


def c_release(table=at(0), max_pages=7, page=16, lens=at(1), ended=at(2), keep=at(3), batch=3, free=at(4), n_pages=9, counts=at(5),
              counts_out=at(6), lens_out=at(7)):
    return _lib.load().tl_release_pages(table, max_pages, page, lens, ended, keep, batch, free, n_pages, counts, counts_out,
                                        lens_out, None)


def c_assign(lens=at(0), new=at(1), batch=3, table=at(2), max_pages=7, page=16, free=at(3), n_pages=9, counts=at(4),
             counts_out=at(5), tokens=5, slots=at(6), positions=at(7), starts=at(8), ends=at(9), ws=at(10), ws_bytes=1 << 20):
    return _lib.load().tl_assign_pages(lens, new, batch, table, max_pages, page, free, n_pages, counts, counts_out, tokens,
                                       slots, positions, starts, ends, ws, ws_bytes, None)


def test_c_pages_refuse():
    odd = ctypes.c_void_p(0x10000008)
    for bad in (dict(table=NULL), dict(lens=NULL), dict(ended=NULL), dict(free=NULL), dict(counts=NULL), dict(counts_out=NULL),
                dict(lens_out=NULL), dict(batch=0), dict(max_pages=0), dict(n_pages=0), dict(page=12), dict(lens_out=at(2)), dict(lens_out=ctypes.c_void_p(at(1).value + 4)),
                dict(counts_out=ctypes.c_void_p(at(5).value + 4)), dict(free=at(0)), dict(counts_out=at(7))):
        assert c_release(**bad) == 1, bad
    for bad in (dict(lens=NULL), dict(new=NULL), dict(table=NULL), dict(free=NULL), dict(counts=NULL), dict(counts_out=NULL),
                dict(slots=NULL), dict(positions=NULL), dict(starts=NULL), dict(ends=NULL), dict(ws=NULL), dict(ws=odd),
                dict(ws_bytes=16), dict(batch=0), dict(max_pages=0), dict(n_pages=0), dict(page=12), dict(tokens=-1),
                dict(ends=at(0)), dict(starts=at(9)), dict(slots=at(7)), dict(table=at(3)),
                dict(counts_out=ctypes.c_void_p(at(4).value + 4))):
        assert c_assign(**bad) == 1, bad
    assert c_release(batch=65536) == c_release(max_pages=1 << 27, batch=1) == 801
    assert c_assign(batch=65536, ws_bytes=1 << 30) == c_assign(max_pages=1 << 27, batch=1) == 801
    assert c_assign(n_pages=1 << 27) == 801


S2, S3 = _lib.strides(512, 64), _lib.strides(512, 64, 64)


def c_slots(q=at(0), qo=at(0), kn=at(16), vn=at(32), kp=at(48), vp=at(64), n_pages=9, page=16, slots=PTR, positions=PTR, cos=None,
            sin=None, rotary=64, n=3, d_k=64, qs=S2, qos=S2, dtype=BF16, kps=S3):
    return _lib.load().tl_paged_kv_append_slots(q, qo, kn, vn, kp, vp, n_pages, page, slots, positions, cos, sin, 9, rotary, 0, n, 4,
                                                2, d_k, qs, qos, S2, S2, kps, S3, dtype, None)


def test_c_append_slots_refuses():
    assert c_slots(n=0) == 0
    for bad in (dict(kn=NULL), dict(vp=NULL), dict(slots=NULL), dict(n_pages=0), dict(page=24), dict(n_pages=1 << 27),
                dict(cos=PTR), dict(cos=PTR, sin=PTR, rotary=66), dict(cos=PTR, sin=PTR, rotary=3), dict(d_k=63),
                dict(cos=PTR, sin=PTR, positions=NULL), dict(dtype=BAD), dict(n=-1), dict(qo=NULL), dict(qs=None), dict(kps=None),
                dict(qos=_lib.strides(512, 128)), dict(qo=ctypes.c_void_p(at(0).value + 128)), dict(qo=at(16)),
                dict(kn=at(48)), dict(qo=at(64)), dict(q=at(48), qo=at(48))):
        assert c_slots(**bad) == 1, bad


def c_packed(q=at(0), table=PTR, lens=PTR, starts=PTR, max_pages=4, n_pages=9, page=16, rows=8, max_new=5, batch=1, heads=(4, 2),
             d_k=64, o=at(16), qs=S2, window=0, dtype=BF16):
    return _lib.load().tl_paged_attention_packed(q, at(32), at(48), table, max_pages, n_pages, page, lens, starts, None, o, None, 0,
                                                 batch, rows, max_new, *heads, d_k, qs, S3, S3, S2, 0.1, window, 0, dtype, None)


def test_c_packed_refuses():
    assert c_packed(batch=0) == c_packed(rows=0) == c_packed(max_new=0) == 0
    for bad in (dict(q=NULL), dict(table=NULL), dict(lens=NULL), dict(starts=NULL), dict(max_pages=0), dict(n_pages=0),
                dict(page=20), dict(max_pages=1 << 27), dict(rows=-1), dict(max_new=-1), dict(heads=(5, 2)), dict(window=-1),
                dict(dtype=BAD), dict(o=at(0)), dict(o=at(32)), dict(qs=None), dict(batch=-1)):
        assert c_packed(**bad) == 1, bad
    for bad in (dict(d_k=96), dict(qs=_lib.strides(512, 68)), dict(q=ctypes.c_void_p(0x100008))):
        assert c_packed(**bad) == 801, bad
    need = _lib.load().tl_paged_packed_workspace_bytes
    padded = _lib.load().tl_paged_prefill_workspace_bytes
    args = (4, 15, 5, 500, 4608, 64, 0, 0, BF16)
    assert need(None, 0, *args) == padded(None, *args) > 0
    assert need(None, 2000, *args) > 0 and need(None, -1, *args) == 0
    # 30 single tokens and 500 rows are no 31 x 500 rows: their keys are divided
    assert need(None, 530, 31, 24, 8, 500, 4096, 128, 0, 0, BF16) > 0 == padded(None, 31, 24, 8, 500, 4096, 128, 0, 0, BF16)


def c_plan(lens=at(0), members=at(1), starts=at(2), shared=at(3), batch=3, groups=2, heads=(4, 2), d_k=64, max_pages=7, page=16,
           dtype=BF16, plan=at(16), nbytes=1 << 30):
    return _lib.load().tl_shared_plan(lens, 0, members, starts, shared, batch, groups, *heads, d_k, max_pages, page, dtype, plan,
                                      nbytes, None)


def c_shared(q=at(0), kp=at(16), vp=at(32), table=PTR, max_pages=7, n_pages=9, page=16, plan=PTR, plan_bytes=1 << 30, groups=2,
             o=at(48), ws=PTR, ws_bytes=1 << 40, batch=3, heads=(4, 2), d_k=64, qs=S2, ks=S3, os=S2, dtype=BF16):
    return _lib.load().tl_paged_attention_shared(q, kp, vp, table, max_pages, n_pages, page, plan, plan_bytes, groups, o, ws,
                                                 ws_bytes, batch, *heads, d_k, qs, ks, S3, os, 0.1, dtype, None)


def test_c_shared_refuses():
    odd = ctypes.c_void_p(0x10000008)
    for bad in (dict(lens=NULL), dict(members=NULL), dict(starts=NULL), dict(shared=NULL), dict(plan=NULL), dict(plan=odd),
                dict(batch=0), dict(groups=0), dict(heads=(5, 2)), dict(heads=(4, 0)), dict(max_pages=0), dict(page=12),
                dict(max_pages=1 << 27), dict(dtype=BAD), dict(nbytes=64), dict(plan=at(2))):
        assert c_plan(**bad) == 1, bad
    for bad in (dict(batch=65536), dict(groups=65536), dict(heads=(129, 1)), dict(d_k=96)):
        assert c_plan(**bad) == 801, bad
    assert c_shared(batch=0) == c_shared(heads=(0, 2)) == 0
    for bad in (dict(q=NULL), dict(table=NULL), dict(plan=NULL), dict(o=NULL), dict(ws=NULL), dict(ws=odd), dict(plan=odd),
                dict(batch=-1), dict(groups=0), dict(heads=(5, 2)), dict(max_pages=0), dict(n_pages=0), dict(page=12),
                dict(max_pages=1 << 27), dict(dtype=BAD), dict(plan_bytes=64), dict(ws_bytes=64), dict(qs=None), dict(o=at(0)), dict(o=at(0), os=_lib.strides(512, 128)),
                dict(o=ctypes.c_void_p(at(0).value + 128)), dict(o=at(16)), dict(o=at(32))):
        assert c_shared(**bad) == 1, bad
    for bad in (dict(batch=65536), dict(groups=65536), dict(heads=(129, 1)), dict(d_k=96), dict(q=odd),
                dict(qs=_lib.strides(512, 68)), dict(ks=_lib.strides(512, 64, 60)), dict(ks=_lib.strides(512, -64, 64)),
                dict(ks=_lib.strides(512, 64, 1 << 25)), dict(os=_lib.strides(-512, 64))):
        assert c_shared(**bad) == 801, bad
    need = _lib.load().tl_shared_plan_bytes
    assert need(0, 1, 4, 2, 64) == need(3, 0, 4, 2, 64) == need(3, 1, 5, 2, 64) == need(3, 1, 4, 2, 32) == 0
    assert need(256, 8, 24, 8, 128) > 0
    assert shared_workspace_bytes(0, 1, 4, 2, 64) == shared_workspace_bytes(3, 1, 129, 1, 64) == 0
    assert shared_workspace_bytes(256, 8, 24, 8, 128) < 1 << 26


# ---- the oracles -----------------------------------------------------------------------

def test_assign_and_release_deal_pages_as_the_host_tables_do():
    """Both take a free list's last page: the same steps give the same tables."""
    rng = np.random.default_rng(0)
    page, batch, n_pages = 4, 5, 40
    host = PageTables(n_pages, page, batch, 32)
    slots = [host.open() for _ in range(batch)]
    table, free = np.full((batch, host.max_pages), -1), np.arange(n_pages - 1, -1, -1)
    counts, lens = [n_pages, 0], np.zeros(batch, np.int64)
    for _ in range(30):
        ended = rng.random(batch) < 0.2
        for b in np.flatnonzero(ended):
            host.close(slots[b])
            slots[b] = host.open()
            assert slots[b] == b
        free, counts, lens = op.release(table, lens, ended, free, counts, page)
        new = np.minimum(rng.integers(0, 6, batch), 32 - lens)
        if new.any():
            host.begin(new)
            host.advance()
        table, places, positions, starts, lens, counts = op.assign(lens, new, table, free, counts, page, 40)
        assert counts == [host.free_pages, 0] and list(lens) == host.lens
        assert free[:counts[0]].tolist() == host._free
        for b in range(batch):
            held = -(-int(lens[b]) // page)
            assert table[b, :held].tolist() == host.tables[b]
            for t in range(starts[b], starts[b + 1]):
                assert positions[t] == lens[b] - new[b] + t - starts[b]
                assert places[t] == host.tables[b][positions[t] // page] * page + positions[t] % page
        assert (places[starts[-1]:] == -1).all()


# ---- which slots share -------------------------------------------------------------------

def test_sharing_follows_forks_writes_and_orders():
    t = PageTables(200, 4, 6, 400)
    a, b = t.open(), t.open()
    t.begin([10, 3, 0, 0, 0, 0])
    t.advance()
    assert t.sharing() == []
    c, d, e = t.fork(a), t.fork(a), t.fork(b)
    assert t.sharing() == [([a, c, d], 3), ([b, e], 1)]
    before = t.version
    t.begin([1, 0, 1, 0, 1, 0])  # a, c and e write: the last pages part
    t.advance()
    assert t.version > before and t.sharing() == [([a, c, d], 2)]
    before = t.version
    for _ in range(3):
        t.begin([0, 1, 0, 0, 0, 0])
        t.advance()
    assert t.version == before
    t.reorder([d], [b])
    assert t.sharing() == [([a, c], 2), ([b, d], 2)]
    t.close(c)
    assert t.sharing() == [([b, d], 2)]
    t.compact()
    assert t.sharing() == [([b, d], 2)]


def test_sharing_of_long_tables():
    t = PageTables(500, 1, 3, 400)
    a = t.open()
    t.begin([100, 0, 0])
    t.advance()
    b, c = t.fork(a), t.fork(a)
    t.begin([1, 1, 0])
    t.advance()
    assert t.sharing() == [([a, b, c], 100)]
    for n in (0, 1, 31, 32, 33, 64, 99):
        t.tables[b][n], keep = -7, t.tables[b][n]
        assert t.sharing() == [([a, c], 100)] if n == 0 else t.sharing() == [([a, b, c], n)]
        t.tables[b][n] = keep


def test_share_reads_goes_without_a_window():
    with pytest.raises(ValueError, match="without a window"):
        PagedKVCache(1, 4, 2, 64, n_pages=4, max_batch=2, max_seq=64, window=16, share_reads=True)
