"""Refusals of the paged cache, windowed attention and beam selection: every call here is refused,
or has nothing to do, before any device work, in the Python layer and at the C entries."""

import ctypes

import numpy as np
import pytest

from triton_llm import _lib, gpu
from triton_llm.kernels import (allocate_kv_pages, beam_select, copy_kv_pages, paged_attention_decode,
                                paged_attention_prefill, paged_decode_workspace, paged_kv_append, window_attention,
                                write_i32)

F32, BF16, BAD = _lib.DTYPE_F32, _lib.DTYPE_BF16, 99


def fake(shape, dtype=np.float32):
    return gpu.DeviceTensor(ctypes.c_void_p(None), shape, dtype, 0, defer_free=False)


def i32(*shape):
    return fake(shape, np.int32)


POOL = (9, 2, 16, 64)


@pytest.mark.parametrize("args,msg", [
    ((0, 2, 16, 64), "positive"), ((4, 0, 16, 64), "positive"), ((4, 2, 16, 0), "positive"),
    ((4, 2, 8, 64), "power of 2"), ((4, 2, 48, 64), "power of 2"), ((4, 2, 2048, 64), "power of 2")])
def test_allocate_refuses(args, msg):
    with pytest.raises(ValueError, match=msg):
        allocate_kv_pages(*args)


def append_args(**change):
    a = dict(q=fake((3, 5, 4, 64)), k=fake((3, 5, 2, 64)), v=fake((3, 5, 2, 64)), kp=fake(POOL), vp=fake(POOL),
             table=i32(3, 7), lens=i32(3), cos=fake((50, 32)), sin=fake((50, 32)))
    a.update(change)
    kw = {n: a.pop(n) for n in ("new_lens", "q_out") if n in a}
    return list(a.values()), kw


@pytest.mark.parametrize("change,msg", [
    ({"kp": fake((9, 2, 16))}, "matching 4-D"),
    ({"vp": fake((9, 2, 32, 64))}, "matching 4-D"),
    ({"kp": fake((9, 2, 24, 64)), "vp": fake((9, 2, 24, 64))}, "power of 2"),
    ({"table": fake((3, 7))}, "page_table must be int32"),
    ({"table": i32(3, 0)}, "page_table must be int32"),
    ({"table": i32(3, 1 << 28)}, "exceed"),
    ({"lens": i32(4)}, "cache_lens must be int32"),
    ({"lens": fake((3,))}, "cache_lens must be int32"),
    ({"k": fake((3, 5, 3, 64))}, "k_new shape"),
    ({"k": fake((5, 128))}, "3-D or 4-D"),
    ({"v": fake((3, 4, 2, 64))}, "v_new shape"),
    ({"q": fake((3, 4, 4, 64))}, "does not match k_new"),
    ({"q": fake((3, 5, 3, 64))}, "multiple of n_kv_head"),
    ({"q": None, "q_out": fake((3, 5, 4, 64))}, "without q_dev"),
    ({"q_out": fake((3, 5, 2, 64))}, "out must be like q"),
    ({"v": fake((3, 5, 2, 64), np.float16)}, "share one dtype"),
    ({"q": fake((3, 5, 4, 64), np.float16)}, "share one dtype"),
    ({"cos": None}, "both be given"),
    ({"cos": fake((50, 33)), "sin": fake((50, 33))}, "cos/sin tables"),
    ({"cos": fake((50, 32), np.float64), "sin": fake((50, 32), np.float64)}, "cos/sin tables"),
    ({"new_lens": i32(2)}, "new_lens must be int32"),
])
def test_append_refuses(change, msg):
    args, kw = append_args(**change)
    with pytest.raises(ValueError, match=msg):
        paged_kv_append(*args, **kw)


@pytest.mark.parametrize("change,msg", [
    ({"n_kv_head": 4}, "KV heads"), ({"n_head": 5}, "multiple of n_kv_head"), ({"n_head": 0}, "multiple"),
    ({"window": -1}, "window and sinks"), ({"sinks": -1}, "window and sinks"), ({"window": 1 << 31}, "window"),
    ({"q": fake((3, 4, 32))}, "q shape"), ({"vp": fake(POOL, np.float16)}, "share one dtype"),
    ({"kp": fake((9, 2, 16, 32)), "vp": fake((9, 2, 16, 32))}, "d_k in"),
    ({"out": fake((3, 4, 32))}, "out must be like q"), ({"lens": i32(2)}, "cache_lens"),
])
def test_decode_and_prefill_refuse(change, msg):
    for shape, call in (((3, 4, 64), paged_attention_decode), ((3, 6, 4, 64), paged_attention_prefill)):
        a = dict(q=fake(shape), kp=fake(POOL), vp=fake(POOL), table=i32(3, 7), lens=i32(3), n_head=4, n_kv_head=2)
        a.update(change)
        kw = {n: a.pop(n) for n in ("window", "sinks", "out") if n in a}
        with pytest.raises(ValueError, match=msg):
            call(*a.values(), **kw)
    with pytest.raises(ValueError, match="exceed"):
        paged_attention_prefill(fake((3, 6, 4, 64)), fake(POOL), fake(POOL), i32(3, 1 << 27), i32(3), 4, 2)
    with pytest.raises(ValueError, match="new_lens"):
        paged_attention_prefill(fake((3, 6, 4, 64)), fake(POOL), fake(POOL), i32(3, 7), i32(3), 4, 2, new_lens=i32(1))
    with pytest.raises(ValueError, match="multiple"):
        paged_decode_workspace(1, 5, 2, 100, 64)


def test_window_refuses():
    q, k = fake((1, 4, 6, 64)), fake((1, 2, 6, 64))
    for args, msg in [((q, k, fake((1, 2, 5, 64)), 4), "expected q"), ((q, fake((2, 2, 6, 64)), fake((2, 2, 6, 64)), 4), "disagree"),
                      ((fake((1, 3, 6, 64)), k, k, 4), "multiple"), ((q, k, k, -1), "window and sinks"),
                      ((q, k, k, 4, -2), "window and sinks"), ((fake((1, 4, 6, 32)), fake((1, 2, 6, 32)), fake((1, 2, 6, 32)), 4), "d_k in")]:
        with pytest.raises(ValueError, match=msg):
            window_attention(*args, out=fake(args[0].shape))
    with pytest.raises(ValueError, match="out shape"):
        window_attention(q, k, k, 4, out=fake((1, 4, 5, 64)))
    with pytest.raises(ValueError, match="seq_k"):
        window_attention(q, fake((1, 2, 0, 64)), fake((1, 2, 0, 64)), 4, out=fake(q.shape))


@pytest.mark.parametrize("src,dst,msg", [
    ([0], [1, 2], "1 source pages, 2"), ([9], [1], r"\[0, 9\)"), ([-1], [1], r"\[0, 9\)"), ([1], [9], r"\[0, 9\)"),
    ([1, 2], [3, 3], "destination twice"), ([1, 2], [2, 3], "source and destination"), ([4], [4], "source and dest")])
def test_copy_refuses(src, dst, msg):
    with pytest.raises(ValueError, match=msg):
        copy_kv_pages([fake(POOL), fake(POOL)], src, dst)


def test_copy_refuses_pools_that_differ():
    with pytest.raises(ValueError, match="pools differ"):
        copy_kv_pages([fake(POOL), fake((9, 2, 16, 32))], [0], [1])
    with pytest.raises(ValueError, match="pools differ"):
        copy_kv_pages([fake(POOL), fake(POOL, np.float16)], [0], [1])
    with pytest.raises(ValueError, match="4-D"):
        copy_kv_pages([fake((9, 16, 32))], [0], [1])
    copy_kv_pages([], [0], [1])
    copy_kv_pages([fake(POOL)], [], [])


def test_write_i32_refuses():
    for index, value, msg in [([0, 1], [2], "2 indices"), ([6], [0], r"\[0, 6\)"), ([-1], [0], r"\[0, 6\)"),
                              ([2, 2], [0, 1], "twice"), ([0], [1 << 31], "int32")]:
        with pytest.raises(ValueError, match=msg):
            write_i32(i32(2, 3), index, value)
    with pytest.raises(ValueError, match="must be int32"):
        write_i32(fake((6,)), [0], [0])
    write_i32(i32(6), [], [])


def test_beam_refuses():
    for logits, scores, n, msg in [
            (fake((6, 100)), fake((2, 3), np.float16), 4, "scores must be float32"),
            (fake((6, 100)), fake((6,)), 4, "scores must be float32"),
            (fake((5, 100)), fake((2, 3)), 4, "do not hold 2 x 3"),
            (fake((6, 0)), fake((2, 3)), 4, "vocab > 0"), (fake((6,)), fake((2, 3)), 4, "vocab > 0"),
            (fake((6, 100), np.int32), fake((2, 3)), 4, "unsupported dtype"),
            (fake((6, 100)), fake((2, 3)), -1, "n_select must be >= 0")]:
        with pytest.raises(ValueError, match=msg):
            beam_select(logits, scores, n)
    out = (fake((2, 4)), i32(2, 4), i32(2, 5))
    with pytest.raises(ValueError, match="out must be"):
        beam_select(fake((6, 100)), fake((2, 3)), 4, out=out)


# ---- the C entries ---------------------------------------------------------------------

NULL, PTR = ctypes.c_void_p(None), ctypes.c_void_p(0x100000)  # PTR is never followed: the calls are refused
S3 = _lib.strides(512, 64, 64)


def c_append(q=PTR, qo=PTR, kn=PTR, table=PTR, max_pages=4, n_pages=9, page=16, cos=None, sin=None, rows=9, rotary=64,
             batch=2, n_new=3, d_k=64, qs=S3, qos=S3, dtype=BF16):
    return _lib.load().tl_paged_kv_append(q, qo, kn, PTR, PTR, PTR, table, max_pages, n_pages, page, PTR, None, cos,
                                          sin, rows, rotary, 0, batch, n_new, 4, 2, d_k, qs, qos, S3, S3, S3, S3,
                                          dtype, None)


def test_c_append_refuses():
    assert c_append(batch=0) == 0 and c_append(n_new=0) == 0
    for bad in (dict(kn=NULL), dict(table=NULL), dict(max_pages=0), dict(n_pages=0), dict(page=24), dict(page=8),
                dict(page=2048), dict(max_pages=1 << 28), dict(cos=PTR), dict(cos=PTR, sin=PTR, rotary=66),
                dict(cos=PTR, sin=PTR, rotary=0), dict(cos=PTR, sin=PTR, rotary=3), dict(d_k=63), dict(dtype=BAD),
                dict(batch=-1), dict(qo=NULL), dict(qs=None), dict(qos=_lib.strides(512, 64, 128)),
                dict(qo=ctypes.c_void_p(0x100010))):
        assert c_append(**bad) == 1, bad


def c_decode(q=PTR, page=16, max_pages=4, window=0, sinks=0, ws=PTR, ws_bytes=1 << 30, batch=2, heads=(4, 2), d_k=64,
             qs=S3, ks=S3, dtype=BF16):
    return _lib.load().tl_paged_attention_decode(q, PTR, PTR, PTR, max_pages, 9, page, PTR, 0, window, sinks, PTR, ws,
                                                 ws_bytes, batch, *heads, d_k, qs, ks, S3, S3, 0.1, dtype, None)


def test_c_decode_refuses():
    assert c_decode(batch=0) == 0
    for bad in (dict(q=NULL), dict(page=12), dict(max_pages=0), dict(max_pages=1 << 27), dict(window=-1),
                dict(sinks=-1), dict(ws=NULL), dict(ws=ctypes.c_void_p(0x100008)), dict(ws_bytes=1000), dict(batch=-1),
                dict(heads=(5, 2)), dict(heads=(4, 0)), dict(dtype=BAD), dict(qs=None)):
        assert c_decode(**bad) == 1, bad
    for bad in (dict(d_k=32), dict(d_k=256), dict(batch=70000), dict(ks=_lib.strides(512, 64, 66)),
                dict(q=ctypes.c_void_p(0x100004)), dict(ks=_lib.strides(512, -64, 64))):
        assert c_decode(**bad) == 801, bad
    ws = _lib.load().tl_paged_decode_workspace_bytes
    tags = 2048 * 2 * 8
    assert ws(24, 8, 128) == tags + 2048 * 2 * 3 * (2 + 128) * 4
    assert ws(16, 1, 64) == tags + 2048 * 2 * 8 * (2 + 64) * 4
    assert ws(0, 1, 64) == ws(5, 2, 64) == ws(4, 2, 0) == 0


def c_window(q=PTR, sq=8, sk=8, heads=(4, 2), d_k=64, qs=S3, ks=S3, window=0, sinks=0, dtype=BF16, batch=1):
    return _lib.load().tl_window_attention(q, PTR, PTR, PTR, None, 0, batch, *heads, sq, sk, d_k, qs, ks, S3, S3, 0.1, window,
                                           sinks, dtype, None)


def c_prefill(table=PTR, lens=PTR, max_pages=4, n_pages=9, page=16, n_new=5, batch=1, **kw):
    q, d_k = kw.get("q", PTR), kw.get("d_k", 64)
    return _lib.load().tl_paged_attention_prefill(q, PTR, PTR, table, max_pages, n_pages, page, lens, None, PTR, None, 0, batch,
                                                  n_new, 4, 2, d_k, S3, S3, S3, S3, 0.1, 0, 0, BF16, None)


def test_c_window_and_prefill_refuse():
    assert c_window(sq=0) == 0 and c_window(batch=0) == 0 and c_prefill(n_new=0) == 0 and c_prefill(batch=0) == 0
    for bad in (dict(q=NULL), dict(sk=0), dict(heads=(3, 2)), dict(window=-1), dict(sinks=-1), dict(dtype=BAD),
                dict(batch=-1), dict(sq=-1), dict(qs=None)):
        assert c_window(**bad) == 1, bad
    for bad in (dict(d_k=32), dict(qs=_lib.strides(512, 64, 68)), dict(ks=_lib.strides(512, 64, 60)),
                dict(q=ctypes.c_void_p(0x100008)), dict(ks=_lib.strides(512, 64, 1 << 25)), dict(sq=1 << 30)):
        assert c_window(**bad) == 801, bad
    for bad in (dict(table=NULL), dict(lens=NULL), dict(max_pages=0), dict(n_pages=0), dict(page=20),
                dict(max_pages=1 << 27), dict(q=NULL)):
        assert c_prefill(**bad) == 1, bad
    assert c_prefill(d_k=96) == 801


def test_c_copy_and_write_refuse():
    lib = _lib.load()
    bases = (ctypes.c_void_p * 2)(0x100000, 0x200000)

    def ints(*x):
        return (ctypes.c_int32 * len(x))(*x)

    def copy(caches=bases, n=2, page=4096, stride=4096, pages=9, src=ints(1, 2), dst=ints(3, 4), count=2):
        return lib.tl_copy_pages(caches, n, page, stride, pages, src, dst, count, None)

    assert copy(n=0) == 0 and copy(count=0) == 0
    for bad in (dict(caches=None), dict(n=-1), dict(page=8), dict(page=4100), dict(stride=2048), dict(stride=4104),
                dict(pages=0), dict(pages=4), dict(src=ints(-1, 2)), dict(dst=ints(3, 9)), dict(src=None), dict(count=-1),
                dict(caches=(ctypes.c_void_p * 2)(0x100000, 0x200008)), dict(caches=(ctypes.c_void_p * 2)(0x100000, None))):
        assert copy(**bad) == 1, bad
    assert copy(page=(1 << 30) + 16, stride=1 << 31) == 801
    assert lib.tl_write_i32(None, 9, None, None, 0, None) == 0
    assert lib.tl_write_i32(None, 9, ints(1), ints(1), 1, None) == 1
    assert lib.tl_write_i32(PTR, 9, ints(9), ints(1), 1, None) == 1
    assert lib.tl_write_i32(PTR, 9, ints(-1), ints(1), 1, None) == 1
    assert lib.tl_write_i32(PTR, 9, ints(1), ints(1), -1, None) == 1


def test_c_beam_refuses():
    lib = _lib.load()

    def beam(logits=PTR, batch=2, beams=4, vocab=100, stride=100, select=8, ws=PTR, ws_bytes=1 << 30, dtype=F32):
        return lib.tl_beam_select(logits, PTR, batch, beams, vocab, stride, select, PTR, PTR, PTR, ws, ws_bytes, dtype,
                                  None)

    assert beam(batch=0) == 0 and beam(select=0) == 0
    for bad in (dict(logits=NULL), dict(batch=-1), dict(beams=0), dict(vocab=0), dict(stride=99), dict(select=-1),
                dict(ws=NULL), dict(ws=ctypes.c_void_p(0x100008)), dict(ws_bytes=16), dict(dtype=BAD)):
        assert beam(**bad) == 1, bad
    for bad in (dict(beams=65), dict(batch=20000), dict(vocab=300000, stride=300000), dict(select=65)):
        assert beam(**bad) == 801, bad
    assert lib.tl_beam_max_select() == 64
    ws = lib.tl_beam_select_workspace_bytes
    assert ws(0, 1, 10) == ws(1, 65, 10) == ws(1, 1, 0) == ws(1, 1, 300000) == 0
    assert ws(2, 4, 128256) >= 8 * 2004 * 4


def test_beam_refuses_sizes_the_kernels_do_not_take():
    for logits, scores, n in [((65, 10), (1, 65), 4), ((4, 300000), (1, 4), 4), ((4, 100), (1, 4), 65),
                              ((80000, 10), (40000, 2), 4)]:
        with pytest.raises(ValueError, match="is not supported"):
            beam_select(fake(logits), fake(scores), n)
