"""PagedKVCache.attention in place of its queries, in steps that share reads and in steps that do not; what it refuses is refused
before the step's tokens are written and the queries turned."""

import numpy as np
import pytest

from oracle import numerics as on
from tests import _paged as P
from triton_llm import gpu
from triton_llm.kernels import precompute_cos_sin
from triton_llm.paged_cache import PagedKVCache

pytestmark = pytest.mark.gpu
HQ, HKV, D, BATCH = 6, 2, 64, 4


def cache_of(dtype, share_reads, prefix):
    """Four slots behind one prompt of `prefix` tokens, one of which rests, in a step that has begun."""
    rng = np.random.default_rng(5)
    cache = PagedKVCache(1, HQ, HKV, D, n_pages=200, max_batch=BATCH, max_seq=1200, dtype=P.H.GPU_DTYPES[dtype],
                         share_reads=share_reads)
    a = cache.open()
    cache.begin([prefix, 0, 0, 0])
    tab = [gpu.to_device(x) for x in precompute_cos_sin(1200, D)]
    cache.attention(0, *(P.dev(P.values(rng, (BATCH, prefix, h, D), dtype), dtype) for h in (HQ, HKV, HKV)), *tab)
    cache.advance()
    for _ in range(BATCH - 1):
        cache.fork(a)
    cache.begin([1, 1, 0, 1])
    rows = [P.values(rng, (BATCH, 1, h, D), dtype) for h in (HQ, HKV, HKV)]
    return cache, rows, tab


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("prefix", [600, 40])
def test_out_is_q(dtype, prefix):
    """As a cache that reads for every slot: the step's sharing does not decide which calls there are."""
    got = []
    for share_reads in (False, True):
        cache, rows, tab = cache_of(dtype, share_reads, prefix)
        assert cache._shares == (share_reads and prefix > 512)
        q, k, v = (P.dev(x, dtype) for x in rows)
        out = cache.attention(0, q, k, v, *tab, out=q)
        assert out is q
        got.append(on.from_storage(P.H.download(out), dtype))
        cache.advance()
    active = [0, 1, 3]
    assert np.isfinite(got[0][active]).all()
    np.testing.assert_array_equal(got[0][active], got[1][active])


@pytest.mark.parametrize("share_reads,prefix", [(False, 40), (True, 40), (True, 600)])
def test_refused_before_anything_changes(share_reads, prefix):
    cache, rows, tab = cache_of("bfloat16", share_reads, prefix)
    q, k, v = (P.dev(x, "bfloat16") for x in rows)
    pools = [gpu.to_host(cache.layers[0][n]) for n in "kv"]
    pool = cache.layers[0]["k"]
    inside = gpu.DeviceTensor(pool.ptr, q.shape, q.dtype, q.nbytes, defer_free=False)
    two = gpu.zeros((BATCH + 1, 1, HQ, D), q.dtype)
    head = gpu.DeviceTensor(two.ptr, q.shape, q.dtype, q.nbytes, defer_free=False)
    tail = gpu.DeviceTensor(type(two.ptr)(two.data_ptr() + 2 * HQ * D), q.shape, q.dtype, q.nbytes, defer_free=False)
    gpu.copy_(head, q)
    for q_in, out in ((q, gpu.zeros((BATCH, HQ, D), q.dtype)), (q, gpu.zeros(q.shape, np.float32)), (q, inside), (head, tail)):
        with pytest.raises(ValueError, match="out"):
            cache.attention(0, q_in, k, v, *tab, out=out)
        np.testing.assert_array_equal(gpu.to_host(q_in), rows[0])
        for n, before in zip("kv", pools):
            np.testing.assert_array_equal(gpu.to_host(cache.layers[0][n]), before)
    want = P.back(cache.attention(0, q, k, v, *tab), "bfloat16")  # the step goes on
    assert np.isfinite(want[[0, 1, 3]]).all()


def test_a_prompt_in_place_is_refused_before_anything_changes():
    cache, _, tab = cache_of("bfloat16", False, 40)
    cache.advance()
    cache.begin([3, 1, 0, 0])
    rng = np.random.default_rng(6)
    rows = [P.values(rng, (BATCH, 3, h, D), "bfloat16") for h in (HQ, HKV, HKV)]
    q, k, v = (P.dev(x, "bfloat16") for x in rows)
    before = gpu.to_host(cache.layers[0]["k"])
    with pytest.raises(ValueError, match="out"):
        cache.attention(0, q, k, v, *tab, out=q)
    np.testing.assert_array_equal(gpu.to_host(q), rows[0])
    np.testing.assert_array_equal(gpu.to_host(cache.layers[0]["k"]), before)
