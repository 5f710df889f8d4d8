"""Prompt attention over padded batches: the work is planned by the rows that there are, not by the longest sequence's for all."""

import ctypes

import numpy as np
import pytest

from oracle import numerics as on
from oracle import paged as op
from tests import _paged as P
from triton_llm import _lib, gpu
from triton_llm.kernels import paged_attention_prefill
from triton_llm.kernels._common import record
from triton_llm.paged_cache import PagedKVCache


def fake(shape, dtype=np.float32):
    return gpu.DeviceTensor(ctypes.c_void_p(None), shape, dtype, 0, defer_free=False)


def workspace(counts, batch, n_new, keys, d_k=128, window=0, dtype=_lib.DTYPE_BF16):
    host = None if counts is None else (ctypes.c_int32 * batch)(*counts)
    return _lib.load().tl_paged_prefill_workspace_bytes(host, batch, 24, 8, n_new, keys, d_k, window, 0, dtype)


def test_padded_batches_are_planned_by_their_rows():
    """One sequence's rows take the plan of a batch of one, whatever the padding; resting sequences count for nothing."""
    alone = workspace(None, 1, 500, 8192)
    assert alone > 0 and workspace(None, 8, 500, 8192) == 0  # by padded rows the device looks full
    assert workspace([0, 0, 0, 500, 0, -3, 0, 0], 8, 500, 8192) == alone
    assert workspace([200] * 2 + [0] * 6, 8, 2000, 8192) == workspace(None, 2, 200, 8192) > 0
    assert workspace([900] * 8, 8, 500, 8192) == workspace(None, 8, 500, 8192)
    assert workspace([0] * 8, 8, 500, 8192) == 0
    for window in (0, 300):
        for d_k in (64, 128):
            assert workspace([500] * 2, 2, 500, 4096, d_k, window) == workspace(None, 2, 500, 4096, d_k, window) == \
                _lib.load().tl_window_workspace_bytes(2, 24, 8, 500, 4096, d_k, window, 0, _lib.DTYPE_BF16)


def test_host_counts_are_checked():
    pool, i32 = fake((9, 2, 16, 64)), lambda *s: fake(s, np.int32)
    args = (fake((3, 6, 4, 64)), pool, pool, i32(3, 7), i32(3), 4, 2)
    for counts, new_lens, msg in [([1, 2, 3], None, "without new_lens"), ([1, 2], i32(3), "must hold 3"),
                                  ([1, 2, 1 << 31], i32(3), "fit in int32"),
                                  ((ctypes.c_int64 * 3)(), i32(3), "int32 numbers"), ((ctypes.c_int32 * 4)(), i32(3), "must hold 3")]:
        with pytest.raises(ValueError, match=msg):
            paged_attention_prefill(*args, new_lens=new_lens, host_new_lens=counts, out=args[0])


# ---- on the GPU ----------------------------------------------------------------------

class Batch:
    """Sequences of lens[b] cached and new[b] new tokens in one pool, q padded to the longest."""

    def __init__(self, dtype, Hq, Hkv, D, lens, new, page=16, seed=0):
        rng = np.random.default_rng(seed)
        self.dtype, self.Hq, self.Hkv, self.D, self.lens, self.new = dtype, Hq, Hkv, D, lens, new
        total = [a + b for a, b in zip(lens, new)]
        pages = sum(-(-n // page) for n in total) + 2
        self.table = P.shuffled_table(rng, total, page, -(-max(total) // page), pages)
        self.q = P.values(rng, (len(lens), max(new), Hq, D), dtype)
        self.kp, self.vp = (P.values(rng, (pages, Hkv, page, D), dtype) for _ in "kv")
        self.dev = [P.dev(x, dtype) for x in (self.q, self.kp, self.vp)] + [P.int32(self.table), P.int32(lens)]

    def run(self, host=None, new=None, out=None, workspace=None):
        """The output as stored, NaN where nothing is written."""
        if out is None:
            out = P.dev(np.full(self.q.shape, on.nan_storage(self.dtype), self.q.dtype), self.dtype)
        paged_attention_prefill(*self.dev, self.Hq, self.Hkv, new_lens=P.int32(self.new if new is None else new), out=out,
                                host_new_lens=host, workspace=workspace)
        gpu.synchronize()
        return P.back(out, self.dtype)

    def check(self, got):
        kf, vf = on.from_storage(self.kp, self.dtype), on.from_storage(self.vp, self.dtype)
        for b, n in enumerate(self.new):
            assert np.isnan(got[b, n:]).all()
            if not n:
                continue
            total = self.lens[b] + n
            k, v = op.gather(kf, self.table[b], total)[0], op.gather(vf, self.table[b], total)[0]
            rows = np.unique(np.r_[0, n - 1, np.linspace(0, n - 1, 9).astype(int)])
            q = np.ascontiguousarray(self.q[b, rows].transpose(1, 0, 2))
            want, tol = P.rows_want(q, k, v, self.lens[b] + rows, True, 0, 0, self.D ** -0.5, self.dtype)
            P.check(f"sequence {b}, {n} rows at {self.lens[b]}", got[b, rows].transpose(1, 0, 2), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,Hq,Hkv,D,prefix,n", [("bfloat16", 24, 8, 128, 4000, 500), ("float16", 15, 5, 64, 3000, 200),
                                                     ("float32", 9, 3, 64, 1500, 130)])
def test_one_of_eight_is_as_alone(dtype, Hq, Hkv, D, prefix, n):
    """The bits of a batch of one: its keys are divided alike.  Without the host's counts they are not."""
    lens, new = [0, 7, 0, prefix, 900, 0, 0, 0], [0, 0, 0, n, 0, 0, 0, 0]
    x = Batch(dtype, Hq, Hkv, D, lens, new)
    got = x.run(new)
    x.check(got)
    x.check(x.run())
    assert (x.run(new)[3] == got[3]).all()
    one = Batch(dtype, Hq, Hkv, D, [prefix], [n])
    one.dev = [gpu.to_device(x.q[3:4], x.dev[0].dtype), *x.dev[1:3], P.int32(x.table[3:4]), P.int32([prefix])]
    one.q = x.q[3:4]
    np.testing.assert_array_equal(one.run([n])[0], got[3])
    np.testing.assert_array_equal(one.run()[0], got[3])


@pytest.mark.gpu
@pytest.mark.parametrize("lens,new", [([0] + [2000] * 7, [300] + [1] * 7), ([900, 0, 50, 1600], [0, 0, 0, 2]), ([5] * 70, [3] * 35 + [0] * 35),
                                      ([10, 4000], [1200, 1]), ([0, 0, 0], [0, 40, 0])])
def test_mixed_steps(lens, new):
    x = Batch("bfloat16", 6, 2, 64, lens, new)
    x.check(x.run(new))
    x.check(x.run((ctypes.c_int32 * len(new))(*new)))


@pytest.mark.gpu
@pytest.mark.parametrize("tiles,parts", [([60] * 17 + [2] * 3, None), ([25] * 13 + [100] + [1] * 6, 5)])
def test_parts_for_two_rounds(monkeypatch, tiles, parts):
    """More parts than workgroups at a time: row tiles stay whole unless one is longer than two parts.  tiles: key tiles of
    sequences of one row tile."""
    P.H.set_override(monkeypatch, "TRITON_LLM_HIP_MAX_CUS", 24)
    slots, n_kv = 3 * 24, 2
    share = int(sum(tiles) * n_kv / (slots // 2) * 1.00001) + 1
    assert slots // 2 < len(tiles) * n_kv < slots < n_kv * sum(-(-t // share) for t in tiles)
    assert (-(-max(tiles) // share) == parts) if max(tiles) > 2 * share else parts is None
    x = Batch("float16", 6, 2, 64, [64 * t - 3 for t in tiles], [2] * len(tiles))
    x.check(x.run(x.new))
    x.check(x.run())


@pytest.mark.gpu
def test_counts_that_are_too_small_reach_nothing_else():
    """More rows on the device than the host said: what is written is right or left, and nothing else is."""
    x = Batch("float16", 6, 2, 64, [900] * 6, [250] * 6)
    told = [1, 0, 0, 0, 0, 0]
    need = _lib.load().tl_paged_prefill_workspace_bytes((ctypes.c_int32 * 6)(*told), 6, 6, 2, 250, x.table.shape[1] * 16, 64, 0, 0,
                                                        _lib.DTYPE_F16)
    assert need > 0
    room = gpu.to_device(np.full(need + (1 << 16), 0xA5, np.uint8))
    ws = gpu.DeviceTensor(ctypes.c_void_p(room.data_ptr()), (need,), room.dtype, need, defer_free=False)
    # the wrapper asks for the larger of both plans' workspaces; the C entry takes what this plan needs
    out = P.dev(np.full(x.q.shape, on.nan_storage(x.dtype), x.q.dtype), x.dtype)
    new = P.int32(x.new)
    s4, page = _lib.strides(250 * 6 * 64, 64, 6 * 64), _lib.strides(2 * 16 * 64, 16 * 64, 64)
    rc = gpu.runtime().tl_paged_attention_prefill_counted(
        *(t.ptr for t in x.dev[:3]), x.dev[3].ptr, x.table.shape[1], x.kp.shape[0], 16, x.dev[4].ptr, new.ptr,
        (ctypes.c_int32 * 6)(*told), out.ptr, ws.ptr, need, 6, 250, 6, 2, 64, s4, page, page, s4, 0.125, 0, 0, _lib.DTYPE_F16, None)
    gpu.synchronize()
    assert rc == 0
    assert (gpu.to_host(room)[need:] == 0xA5).all()
    got, want = P.back(out, x.dtype), x.run()
    left = np.isnan(got)
    assert left.any() and not left.all()
    # either is within 2^-11 (W + |o|) of the exact output, W = sum p |v| < 1 and |o| < 1 over 900 normal values and more
    np.testing.assert_allclose(got[~left], want[~left], atol=4 * 2.0 ** -11)


@pytest.mark.gpu
def test_recorded_and_captured_steps_follow_the_counts():
    """PagedKVCache's attention, replayed for a step whose prompt is another slot's.  Keys may be divided otherwise: two sums of
    up to 700 terms, each within 2 (700 + 64) 2^-24 + 120 2^-23 of W < 1.5."""
    Hq, Hkv, D, B, n = 12, 4, 64, 8, 220
    c = PagedKVCache(1, Hq, Hkv, D, n_pages=400, max_batch=B, max_seq=1024)
    rng = np.random.default_rng(2)
    for _ in range(B):
        c.open()
    c.begin([300] * B)
    first = [P.dev(P.values(rng, (B, 300, h, D), "float32"), "float32") for h in (Hq, Hkv, Hkv)]
    c.attention(0, *first)
    c.advance()
    x = [P.dev(P.values(rng, (B, n, h, D), "float32"), "float32") for h in (Hq, Hkv, Hkv)]
    out = gpu.zeros((B, n, Hq, D))
    c.begin([n] + [0] * (B - 1))
    gpu.synchronize()
    step = record(lambda: c.attention(0, *x, out=out))
    with gpu.capture() as g:
        c.attention(0, *x, out=out)
    step()
    c.advance()
    for new in ([0, 0, n, 1, 0, 0, 0, 0], [1, 50, 0, 0, 0, 0, 0, n], [40] * B):
        c.begin(new)
        want = gpu.to_host(c.attention(0, *x))
        for replay in (step, g.replay):
            out.from_numpy(np.full(out.shape, np.nan, np.float32))
            replay()
            got = gpu.to_host(out)
            for b, m in enumerate(new):
                np.testing.assert_allclose(got[b, :m], want[b, :m], atol=3.2e-4)
        c.advance()
