"""Weights far below a row's largest in 16-bit windowed and paged attention: many of them together carry the output."""

import numpy as np
import pytest

from oracle import numerics as on
from tests import _paged as P
from triton_llm import gpu
from triton_llm.kernels import paged_attention_prefill, window_attention

pytestmark = pytest.mark.gpu


def flat_tail(D, Sq, Sk, below, dtype):
    """q, k, v of one head whose row sees one key with the largest score (v 0) and, `below` under it, all others
    (v 1 but in its last feature): out = n w / (1 + n w), w = exp(-below).  Scores are exact in 16 bits."""
    q, k, v = np.zeros((1, 1, Sq, D)), np.zeros((1, 1, Sk, D)), np.ones((1, 1, Sk, D))
    q[..., 0] = q[..., 1] = 1
    k[..., 0] = 16 - np.floor(below)
    k[..., 1] = -(below - np.floor(below))
    k[..., 0, :2] = 16, 0
    v[..., 0, :] = 0
    v[..., 1:, -1] = np.arange(Sk - 1) % 7 - 3
    return [on.to_storage(x.astype(np.float32), dtype) for x in (q, k, v)]


@pytest.mark.parametrize("below", [14.5, 16.25])  # weights of 2^-20.9 and 2^-23.4: subnormal in fp16 as they are
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_flat_tail(dtype, D, below):
    Sq, Sk = 3, 6000
    q, k, v = flat_tail(D, Sq, Sk, below, dtype)
    got = P.back(window_attention(*(P.dev(x, dtype) for x in (q, k, v)), 0, sm_scale=1.0), dtype)
    want, tol = P.rows_want(q[0], on.from_storage(k[0], dtype), on.from_storage(v[0], dtype), Sk - Sq + np.arange(Sq), True,
                            0, 0, 1.0, dtype)
    P.check(f"flat tail {dtype} d{D} {below}", got[0], want, tol)


@pytest.mark.parametrize("rise", [2.5, 3.0, 5.5, 6.0, 11.0])
def test_maximum_that_rises(rise):
    """A row's largest score rises from tile to tile by less and by more than what moves the running maximum."""
    D, Sk, dtype = 64, 64 * 9, "float16"
    rng = np.random.default_rng(3)
    q, k, v = (np.zeros(s, np.float32) for s in [(1, 1, 2, D), (1, 1, Sk, D), (1, 1, Sk, D)])
    q[..., 0] = 1
    k[0, 0, :, 0] = -40 + rise * (np.arange(Sk) // 64) + rng.integers(-8, 1, Sk) / 8
    v[:] = rng.standard_normal(v.shape)
    q, k, v = (on.to_storage(x, dtype) for x in (q, k, v))
    got = P.back(window_attention(*(P.dev(x, dtype) for x in (q, k, v)), 0, sm_scale=1.0), dtype)
    want, tol = P.rows_want(q[0], on.from_storage(k[0], dtype), on.from_storage(v[0], dtype), Sk - 2 + np.arange(2), True,
                            0, 0, 1.0, dtype)
    P.check(f"rise {rise}", got[0], want, tol)


def test_flat_tail_in_pages():
    D, Sk, page, dtype = 64, 4000, 32, "float16"
    q, k, v = flat_tail(D, 2, Sk, 14.5, dtype)
    n = Sk // page
    pool = [np.ascontiguousarray(x[0].reshape(1, n, page, D).transpose(1, 0, 2, 3)) for x in (k, v)]
    order = np.random.default_rng(5).permutation(n)
    kp, vp = (np.empty_like(x) for x in pool)
    kp[order], vp[order] = pool
    rows = np.ascontiguousarray(q.transpose(0, 2, 1, 3))
    out = paged_attention_prefill(P.dev(rows, dtype), P.dev(kp, dtype), P.dev(vp, dtype), P.int32(order[None]),
                                  P.int32([Sk - 2]), 1, 1, sm_scale=1.0)
    gpu.synchronize()
    want, tol = P.rows_want(q[0], on.from_storage(k[0], dtype), on.from_storage(v[0], dtype), Sk - 2 + np.arange(2), True,
                            0, 0, 1.0, dtype)
    P.check("flat tail in pages", P.back(out, dtype)[0].transpose(1, 0, 2), want, tol)
