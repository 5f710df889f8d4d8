"""paged_attention_packed's max_new where it is no bound: any number from the rows of q on says the same."""

import sys

import numpy as np
import pytest

from tests import _paged as P
from triton_llm.kernels import paged_attention_packed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_new", [30, 31, 1000, (1 << 31) - 1, 1 << 31, 1 << 32, (1 << 32) + 1, sys.maxsize, np.int64(1 << 40)])
def test_max_new_past_the_rows(max_new):
    rng = np.random.default_rng(4)
    Hq, Hkv, D, page, rows = 4, 2, 64, 16, 30
    kp, vp = (P.dev(P.values(rng, (12, Hkv, page, D), "float16"), "float16") for _ in "kv")
    q = P.dev(P.values(rng, (rows, Hq, D), "float16"), "float16")
    table, lens, starts = P.int32([[0, 1, 2, 3], [4, 5, 6, 7], [8, 9, 10, 11]]), P.int32([3, 40, 17]), P.int32([0, 1, 24, rows])
    got = []
    for n in (rows, max_new):
        out = P.dev(np.zeros((rows, Hq, D), np.float16), "float16")
        got.append(P.back(paged_attention_packed(q, kp, vp, table, lens, starts, Hq, Hkv, n, out=out), "float16"))
    assert got[0].any((1, 2)).all()
    np.testing.assert_array_equal(got[0], got[1])
