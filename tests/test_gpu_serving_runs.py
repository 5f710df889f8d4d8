"""The operators together as programs use them: a server whose page tables the GPU keeps, with packed batches and shared
prefixes; the paged cache with reads shared.  Every step's outputs against attention over every sequence's whole history in 64
bits."""

import numpy as np
import pytest

from oracle import numerics as on
from oracle import paged as op
from tests import _paged as P
from tests.test_gpu_paged_cache import Run
from triton_llm import gpu
from triton_llm.kernels import (allocate_kv_pages, assign_kv_pages, paged_attention_packed, paged_attention_shared,
                                paged_kv_append_slots, plan_shared_attention, precompute_cos_sin, release_kv_pages)
from triton_llm.paged_cache import PagedKVCache

pytestmark = pytest.mark.gpu


class Server:
    """Tables, lengths and the free list on the device; the host keeps every sequence's rotated k and v, and asks for nothing
    else."""

    def __init__(self, dtype, Hq, Hkv, D, page, batch, max_pages, n_pages, tokens):
        self.dtype, self.Hq, self.Hkv, self.D, self.page, self.batch, self.tokens = dtype, Hq, Hkv, D, page, batch, tokens
        self.kp, self.vp = allocate_kv_pages(n_pages, Hkv, page, D, P.H.GPU_DTYPES[dtype])
        self.table = P.int32(np.full((batch, max_pages), -1))
        self.free, self.counts = P.int32(np.arange(n_pages)), P.int32([n_pages, 0])
        self.lens, self.new, self.ended = (gpu.zeros((batch,), np.int32) for _ in range(3))
        self.keep = gpu.zeros((batch,), np.int32)
        self.out = tuple(gpu.zeros((n,), np.int32) for n in (tokens, tokens, batch + 1, batch))
        self.cos, self.sin = precompute_cos_sin(max_pages * page, D)
        self.tab = [gpu.to_device(x) for x in (self.cos, self.sin)]
        self.rows = [gpu.zeros((tokens, h, D), P.H.GPU_DTYPES[dtype]) for h in (Hq, Hkv, Hkv)]
        self.o = gpu.zeros((tokens, Hq, D), P.H.GPU_DTYPES[dtype])
        self.hist = [([], []) for _ in range(batch)]
        self.rng = np.random.default_rng(3)

    def device_step(self, attend):
        """What a captured step holds: nothing in it comes from the host."""
        release_kv_pages(self.table, self.lens, self.ended, self.free, self.counts, self.page, keep=self.keep)
        assign_kv_pages(self.lens, self.new, self.table, self.free, self.counts, self.page, self.tokens, out=self.out)
        slots, positions, starts, ends = self.out
        paged_kv_append_slots(*self.rows, self.kp, self.vp, slots, positions, *self.tab)
        attend(starts, ends)
        gpu.copy_(self.lens, ends)

    def packed(self, starts, ends):
        paged_attention_packed(self.rows[0], self.kp, self.vp, self.table, self.lens, starts, self.Hq, self.Hkv, self.tokens,
                               out=self.o)

    def load(self, new, ended=None):
        """The host's part of a step: counts and the rows' q, k, v, which it remembers."""
        ended = [0] * self.batch if ended is None else ended
        self.new.from_numpy(np.asarray(new, np.int32)), self.ended.from_numpy(np.asarray(ended, np.int32))
        self.now = [P.values(self.rng, (self.tokens, h, self.D), self.dtype) for h in (self.Hq, self.Hkv, self.Hkv)]
        for t, x in zip(self.rows, self.now):
            gpu.copy_(t, P.dev(x, self.dtype))
        self.expect = list(new)
        for b, e in enumerate(ended):
            if e:
                self.hist[b] = ([], [])

    def turn(self, x, pos):
        c, s = self.cos[pos][:, None], self.sin[pos][:, None]
        return on.to_storage(on.round_to(op.rotate(on.from_storage(x, self.dtype), c, s, False), self.dtype), self.dtype)

    def check(self, name):
        got, at = P.back(self.o, self.dtype), 0
        for b, m in enumerate(self.expect):
            if m == 0:
                continue
            q, k, v = (x[at:at + m] for x in self.now)
            hk, hv = self.hist[b]
            pos = len(hk) + np.arange(m)
            hk.extend(self.turn(k, pos))
            hv.extend(v)
            kf, vf = (on.from_storage(np.stack(x), self.dtype).astype(np.float64).transpose(1, 0, 2) for x in (hk, hv))
            qr = np.ascontiguousarray(self.turn(q, pos).transpose(1, 0, 2))
            want, tol = P.rows_want(qr, kf, vf, pos, True, 0, 0, self.D ** -0.5, self.dtype)
            P.check(f"{name} sequence {b} at {pos[0]}", got[at:at + m].transpose(1, 0, 2), want, tol)
            at += m


@pytest.mark.parametrize("dtype,Hq,Hkv,D,page", [("float32", 3, 1, 64, 16), ("bfloat16", 6, 2, 128, 32), ("float16", 4, 4, 64, 16)])
def test_packed_steps(dtype, Hq, Hkv, D, page):
    """Prompts, tokens and ends in packed batches, captured once and replayed with other counts."""
    s = Server(dtype, Hq, Hkv, D, page, batch=6, max_pages=12, n_pages=50, tokens=150)
    s.load([40, 0, 17, 0, 0, 3])
    s.device_step(s.packed)
    s.check("eager")
    s.load([1, 50, 1, 0, 0, 1])
    with gpu.capture() as graph:
        s.device_step(s.packed)
    graph.replay()
    s.check("replay")
    for turn in range(5):
        ended = (s.rng.random(6) < 0.25).astype(int)
        new = np.where(ended, s.rng.integers(0, 2) * s.rng.integers(1, 40, 6), s.rng.integers(0, 3, 6))
        s.load(new.tolist(), ended.tolist())
        graph.replay() if turn % 2 else s.device_step(s.packed)
        s.check(f"turn {turn}")
    s.load([0] * 6, [1] * 6)
    graph.replay()
    assert gpu.to_host(s.counts).tolist() == [50, 0] and sorted(gpu.to_host(s.free).tolist()) == list(range(50))


@pytest.mark.parametrize("dtype,Hq,Hkv,D,page", [("float32", 3, 1, 64, 16), ("bfloat16", 6, 2, 128, 16), ("float16", 12, 2, 64, 32)])
def test_tokens_behind_a_shared_prompt(dtype, Hq, Hkv, D, page):
    """One prompt's pages stand first in every sequence's row; they are read once a step, and stay when sequences end."""
    batch, full = 5, 3
    s = Server(dtype, Hq, Hkv, D, page, batch=batch, max_pages=8, n_pages=40, tokens=full * page)
    s.load([full * page, 0, 0, 0, 0])
    s.device_step(s.packed)
    s.check("prompt")
    # the others begin with its pages: entries, lengths, and how many leading pages are not theirs alone
    table, lens = gpu.to_host(s.table), np.full(batch, full * page, np.int32)
    table[1:, :full] = table[0, :full]
    s.table.from_numpy(table), s.lens.from_numpy(lens), s.keep.from_numpy(np.full(batch, full, np.int32))
    for b in range(1, batch):
        s.hist[b] = tuple(list(x) for x in s.hist[0])
    members, starts, shared = P.int32(np.arange(batch)[::-1]), P.int32([0, batch]), P.int32([full * page])
    state = {"plan": None}

    def attend(_, ends):
        # every sequence has one token: the packed rows are the sequences'
        state["plan"] = plan_shared_attention(s.table, ends, members, starts, shared, Hq, Hkv, D, page, P.H.GPU_DTYPES[dtype],
                                              plan=state["plan"])
        n = batch * Hq * D * s.o.dtype.itemsize
        q, o = (gpu.DeviceTensor(t.ptr, (batch, Hq, D), t.dtype, n, defer_free=False) for t in (s.rows[0], s.o))
        paged_attention_shared(q, s.kp, s.vp, s.table, state["plan"], Hq, Hkv, out=o)

    s.load([1] * batch)
    s.device_step(attend)
    s.check("first tokens")
    s.load([1] * batch)
    with gpu.capture() as graph:
        s.device_step(attend)
    for turn in range(page + 2):  # over the end of a page
        if turn:
            s.load([1] * batch)
        graph.replay()
        s.check(f"turn {turn}")
    s.load([0] * batch, [1] * batch)
    s.device_step(lambda *_: None)
    assert gpu.to_host(s.counts).tolist() == [40 - full, 0]  # the prompt's pages are still held


@pytest.fixture
def every_shared_page(monkeypatch):
    monkeypatch.setattr(PagedKVCache, "SHARE_LEAST", 1)


@pytest.mark.parametrize("dtype,Hq,Hkv,D,page", [("float32", 3, 1, 64, 16), ("bfloat16", 6, 2, 128, 32), ("float16", 20, 1, 64, 16)])
def test_paged_cache_shares_reads(every_shared_page, dtype, Hq, Hkv, D, page):
    """Forks, two groups, slots that rest, copies on write, reorder, compaction: steps of one token go by what is shared then."""
    r = Run(dtype, Hq, Hkv, D, batch=7, n_pages=90, max_seq=300, page_size=page, share_reads=True)
    a, b = r.open(), r.open()
    r.step([70, 65, 0, 0, 0, 0, 0])
    r.step([1, 1, 0, 0, 0, 0, 0])           # nothing is shared
    assert not r.cache._shares
    c, d, e, f = r.fork(a), r.fork(a), r.fork(b), r.fork(b)
    r.step([1, 1, 1, 0, 1, 1, 0])            # a slot of a group rests; last pages are copied
    assert r.cache._shares
    r.step([1, 1, 1, 1, 1, 1, 0])
    r.step([5, 1, 1, 1, 0, 1, 0])            # not one token each: the prompt's path
    assert not r.cache._shares
    g = r.open()
    r.step([1, 1, 1, 1, 1, 1, 1])
    r.reorder([a, c, e], [b, d, e])
    r.step([1, 1, 1, 1, 1, 1, 1])
    r.cache.compact()
    r.step([1, 0, 1, 1, 1, 1, 1])
    for s in (c, d):
        r.cache.close(s)
        del r.hist[s]
    r.step([1, 1, 0, 0, 1, 1, 1])
    assert r.cache._shares
    for s in (a, b, e, f, g):
        r.cache.close(s)
    assert r.cache.free_pages == 90


def test_paged_cache_recorded_while_it_shares(every_shared_page):
    """A layer's call, recorded while slots share, replayed after most of them have ended and nothing is shared any more."""
    Hq, Hkv, D, batch = 4, 2, 64, 4
    r = Run("bfloat16", Hq, Hkv, D, batch=batch, n_layer=1, n_pages=60, max_seq=200, share_reads=True)
    a = r.open()
    r.step([70, 0, 0, 0])
    others = [r.fork(a) for _ in range(3)]
    q_d, k_d, v_d, out = (P.dev(np.zeros((batch, 1, h, D), np.uint16), "bfloat16") for h in (Hq, Hkv, Hkv, Hq))
    attention = r.cache.attention
    graph = None

    def recorded(layer, q, k, v, *tab):
        nonlocal graph
        for to, x in ((q_d, q), (k_d, k), (v_d, v)):
            gpu.copy_(to, x)
        if graph is None:
            with gpu.capture() as graph:
                attention(layer, q_d, k_d, v_d, *tab, out=out)
        graph.replay()
        return out

    r.cache.attention = recorded
    r.step([1, 1, 1, 1])
    assert r.cache._shares
    r.step([1, 1, 0, 1])
    for s in others:
        r.cache.close(s)
        del r.hist[s]
    r.step([1, 0, 0, 0])
    assert not r.cache._shares
    b = r.open()
    r.step([1, 1, 0, 0])
    r.cache.close(a)
    del r.hist[a]
    r.step([0, 1, 0, 0])
    r.fork(b)
    r.step([1, 1, 0, 0])


def test_paged_cache_reads_short_prefixes_each():
    r = Run("bfloat16", 4, 2, 64, batch=3, n_layer=1, n_pages=60, max_seq=400, share_reads=True)
    a = r.open()
    r.step([100, 0, 0])
    r.fork(a), r.fork(a)
    r.step([1, 1, 1])
    assert not r.cache._shares


def test_paged_cache_shares_a_long_prefix():
    r = Run("bfloat16", 4, 2, 64, batch=3, n_layer=1, n_pages=300, max_seq=1400, share_reads=True)
    a = r.open()
    r.step([1050, 0, 0])
    r.fork(a), r.fork(a)
    r.step([1, 1, 1])
    assert r.cache._shares
    r.step([1, 1, 1])
