"""Steps in which slots rest: what rests is not read."""

import ctypes

import numpy as np
import pytest

from tests import _paged as P
from triton_llm import gpu
from triton_llm.paged_cache import PagedKVCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,length", [(4, 40), (6, 900), (3, 5000)])  # a workgroup a sequence, and shares
@pytest.mark.parametrize("new", [1, 3])
def test_resting_slots_are_not_read(batch, length, new):
    """Their pages hold NaN: in a one-token step their rows are zeros, the others' what they are without the NaN."""
    Hq, Hkv, D = 6, 2, 64
    c = PagedKVCache(1, Hq, Hkv, D, n_pages=batch * (length // 16 + 2), max_batch=batch, max_seq=length + 16)
    rng = np.random.default_rng(batch)
    for _ in range(batch):
        c.open()
    c.begin([length] * batch)
    c.attention(0, *(P.dev(P.values(rng, (batch, length, h, D), "float32"), "float32") for h in (Hq, Hkv, Hkv)))
    c.advance()
    step = [0 if s % 2 else new for s in range(batch)]
    x = [P.values(rng, (batch, new, h, D), "float32") for h in (Hq, Hkv, Hkv)]
    c.begin([new] * batch)
    want = gpu.to_host(c.attention(0, *(P.dev(t, "float32") for t in x)))
    # the same step again, from the cache before it, with every second slot at rest
    c.tables.new = [0] * batch
    c.begin(step)
    for s in range(1, batch, 2):
        for page in c.tables.tables[s]:
            for pool in c.layers[0].values():
                n = pool.nbytes // pool.shape[0]
                view = gpu.DeviceTensor(ctypes.c_void_p(pool.data_ptr() + page * n), pool.shape[1:], np.float32, n,
                                        defer_free=False)
                view.from_numpy(np.full(pool.shape[1:], np.nan, np.float32))
    got = gpu.to_host(c.attention(0, *(P.dev(t, "float32") for t in x)))
    for s in range(batch):
        if step[s]:
            # divided among other parts than before: two sums of `length` terms, of W = sum p |v| < 2
            np.testing.assert_allclose(got[s], want[s], atol=4 * (2 * (length + 64) * 2.0 ** -24 + 60 * 2.0 ** -22))
        elif new == 1:
            assert (got[s] == 0).all()
    c.advance()
    assert c.lens == [length + n for n in step]


def test_rest_and_wake():
    """A slot that rested goes on where it was."""
    Hq, Hkv, D, B = 3, 1, 64, 3
    rng = np.random.default_rng(5)
    rows = [[P.values(rng, (B, 1, h, D), "float32") for h in (Hq, Hkv, Hkv)] for _ in range(6)]
    outs = []
    for rests in (False, True):
        c = PagedKVCache(1, Hq, Hkv, D, n_pages=12, max_batch=B, max_seq=64)
        for _ in range(B):
            c.open()
        got = []
        for i, x in enumerate(rows):
            if rests and i % 2:  # a step of slot 1 alone, which is taken back
                c.begin([0, 1, 0])
                c.attention(0, *(P.dev(t, "float32") for t in x))
                c.tables.new = [0] * B
            c.begin([1] * B)
            got.append(gpu.to_host(c.attention(0, *(P.dev(t, "float32") for t in x))))
            c.advance()
        outs.append(np.stack(got))
    np.testing.assert_array_equal(outs[0], outs[1])
