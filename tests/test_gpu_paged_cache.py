"""The paged operators together as a program uses them: prompts, shared prefixes, beam search, windows, compaction,
each step's outputs against attention over every sequence's whole history in 64 bits."""

import numpy as np
import pytest

from oracle import numerics as on
from oracle import paged as op
from tests import _paged as P
from triton_llm import gpu
from triton_llm.kernels import beam_select, gemm, precompute_cos_sin
from triton_llm.paged_cache import PagedKVCache

pytestmark = pytest.mark.gpu


class Run:
    """A cache and, for every slot, the rotated k and the v of its tokens as storage."""

    def __init__(self, dtype, Hq, Hkv, D, batch, n_layer=2, **kw):
        self.dtype, self.Hq, self.Hkv, self.D, self.batch = dtype, Hq, Hkv, D, batch
        self.cache = PagedKVCache(n_layer, Hq, Hkv, D, max_batch=batch, dtype=P.H.GPU_DTYPES[dtype], **kw)
        self.n_layer = n_layer
        self.window, self.sinks = kw.get("window", 0), kw.get("sinks", 0)
        self.cos, self.sin = precompute_cos_sin(kw["max_seq"], D)
        self.tab = [gpu.to_device(x) for x in (self.cos, self.sin)]
        self.hist = {}
        self.rng = np.random.default_rng(1)

    def turn(self, x, pos):
        c, s = self.cos[pos][:, None], self.sin[pos][:, None]
        return on.to_storage(on.round_to(op.rotate(on.from_storage(x, self.dtype), c, s, False), self.dtype), self.dtype)

    def step(self, new, q_of=None):
        """One step of every layer with random rows; checks and returns the last layer's output (batch, n, Hq, D)."""
        n = max(new)
        self.cache.begin(new)
        got = None
        for layer in range(self.n_layer):
            q, k, v = (P.values(self.rng, (self.batch, n, h, self.D), self.dtype) for h in (self.Hq, self.Hkv, self.Hkv))
            out = self.cache.attention(layer, P.dev(q, self.dtype), P.dev(k, self.dtype), P.dev(v, self.dtype), *self.tab)
            got = P.back(out, self.dtype)
            for s, m in enumerate(new):
                if not m:
                    continue
                hk, hv = self.hist[s][layer]
                pos = len(hk) + np.arange(m)
                hk.extend(self.turn(k[s, :m], pos))
                hv.extend(v[s, :m])
                kf, vf = (on.from_storage(np.stack(x), self.dtype).astype(np.float64).transpose(1, 0, 2) for x in (hk, hv))
                qr = self.turn(q[s, :m], pos).transpose(1, 0, 2)
                want, tol = P.rows_want(np.ascontiguousarray(qr), kf, vf, pos, True, self.window, self.sinks, self.D ** -0.5, self.dtype)
                P.check(f"slot {s} layer {layer} at {pos[0]}", got[s, :m].transpose(1, 0, 2), want, tol)
        self.cache.advance()
        return out

    def open(self):
        s = self.cache.open()
        self.hist[s] = [([], []) for _ in range(self.n_layer)]
        return s

    def copy_hist(self, a):
        return [(list(k), list(v)) for k, v in self.hist[a]]

    def fork(self, a):
        s = self.cache.fork(a)
        self.hist[s] = self.copy_hist(a)
        return s

    def reorder(self, slots, parents):
        self.cache.reorder(slots, parents)
        taken = [self.copy_hist(p) for p in parents]
        for s, h in zip(slots, taken):
            self.hist[s] = h


@pytest.mark.parametrize("dtype,Hq,Hkv,D,page,window,sinks", [("float32", 3, 1, 64, 16, 0, 0), ("bfloat16", 6, 2, 128, 32, 0, 0),
                                                              ("float16", 4, 4, 64, 16, 40, 4)])
def test_serving(dtype, Hq, Hkv, D, page, window, sinks):
    r = Run(dtype, Hq, Hkv, D, batch=5, n_pages=60, max_seq=300, page_size=page, window=window, sinks=sinks)
    a, b = r.open(), r.open()
    r.step([50, 17, 0, 0, 0])            # two prompts
    r.step([1, 1, 0, 0, 0])
    c = r.fork(a)                        # a shared prefix, then different questions
    d = r.open()
    r.step([30, 1, 7, 3, 0])
    for _ in range(3):
        r.step([1, 1, 1, 1, 0])
    r.cache.close(b)
    del r.hist[b]
    assert r.cache.compact() >= 0
    r.step([1, 0, 1, 1, 0])
    e = r.fork(c)
    assert e == b  # the lowest closed slot
    r.step([1, 1, 1, 1, 0])
    r.reorder([a, c, d, e], [c, c, e, a])
    r.cache.compact()
    r.step([1, 2, 70, 1, 0])
    for s in (a, c, d, e):
        r.cache.close(s)
    assert r.cache.free_pages == 60


def test_beam_search():
    """Two beam searches of four beams: prefix, forks, then steps of attention, projection, selection and reordering."""
    J, V, dtype = 4, 500, "float32"
    r = Run(dtype, 6, 2, 64, batch=2 * J, n_layer=1, n_pages=80, max_seq=200)
    first = [r.open() for _ in range(2 * J)]
    new = [0] * (2 * J)
    new[0], new[J] = 33, 20
    r.step(new)
    for item in range(2):
        group = first[item * J:(item + 1) * J]
        r.reorder(group, [group[0]] * J)
    w = P.dev(np.random.default_rng(7).standard_normal((6 * 64, V)).astype(np.float32) * 4, dtype)
    scores = np.array([[0] + [-np.inf] * (J - 1)] * 2, np.float32)  # the beams start alike: one counts
    for _ in range(6):
        out = r.step([1] * (2 * J))
        logits = gemm(gpu.view(out, (2 * J, 6 * 64)), w)
        got = [gpu.to_host(t) for t in beam_select(logits, gpu.to_device(scores), J)]
        want = op.beam_select(gpu.to_host(logits).reshape(2, J, V), scores, J)
        np.testing.assert_array_equal(got[1], want[1])
        np.testing.assert_array_equal(got[2], want[2])
        np.testing.assert_allclose(got[0], want[0], rtol=1e-6)
        scores = got[0]
        r.reorder(first, [item * J + int(p) for item in range(2) for p in got[1][item]])
    held = 80 - r.cache.free_pages
    assert held < 2 * J * 4  # the beams share their prefixes


def test_attention_refuses():
    c = PagedKVCache(1, 4, 2, 64, n_pages=8, max_batch=2, max_seq=64)
    q, k = gpu.zeros((2, 3, 4, 64)), gpu.zeros((2, 3, 2, 64))
    with pytest.raises(ValueError, match="begin"):
        c.attention(0, q, k, k)
    c.open()
    c.begin([3, 0])
    for args, msg in [((1, q, k, k), "layer 1"), ((0, k, k, k), "q must be"), ((0, q, q, k), "k must be"),
                      ((0, gpu.zeros((2, 2, 4, 64)), gpu.zeros((2, 2, 2, 64)), gpu.zeros((2, 2, 2, 64))), "2 rows a slot"),
                      ((0, q, k, k, gpu.zeros((2, 32)), gpu.zeros((2, 32))), "exceed the cos/sin table")]:
        with pytest.raises(ValueError, match=msg):
            c.attention(*args)
    with pytest.raises(ValueError, match="share one dtype"):
        c.attention(0, gpu.zeros((2, 3, 4, 64), np.float16), k, k)
