"""An infinity in a V row that a query sees: its feature is not finite, as in the 64-bit form, and no other feature and no sequence that
does not see the row is touched.  Few rows and many, whose weights are multiplied in two words."""

import numpy as np
import pytest

from oracle import numerics as on
from tests import _paged as P
from triton_llm.kernels import paged_attention_packed, paged_attention_shared, plan_shared_attention

pytestmark = pytest.mark.gpu
D, PAGE = 64, 16


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("batch", [4, 40])
def test_shared(dtype, batch):
    """One in the shared part, one in a sequence's own part."""
    rng = np.random.default_rng(31)
    Hq, Hkv, shared = 3, 1, 48
    lens = shared + rng.integers(1, 30, batch)
    table = P.shuffled_table(rng, lens, PAGE, 5, 5 * batch)
    table[1:, :3] = table[0, :3]
    kp, vp = (rng.standard_normal((5 * batch, Hkv, PAGE, D)).astype(np.float32) for _ in "kv")
    q = P.values(rng, (batch, Hq, D), dtype)
    clean = [on.to_storage(x, dtype) for x in (kp, vp)]
    vp[table[0, 1], 0, 5, 7] = np.inf
    vp[table[2, 3], 0, 0, 9] = -np.inf
    k, v = (on.to_storage(x, dtype) for x in (kp, vp))
    plan = plan_shared_attention(P.int32(table), P.int32(lens), P.int32(np.arange(batch)), P.int32([0, batch]), P.int32([shared]), Hq,
                                 Hkv, D, PAGE, P.H.GPU_DTYPES[dtype])
    got = P.back(paged_attention_shared(P.dev(q, dtype), P.dev(k, dtype), P.dev(v, dtype), P.int32(table), plan, Hq, Hkv), dtype)
    assert not np.isfinite(got[..., 7]).any() and not np.isfinite(got[2, :, 9]).any()
    want, tol = P.decode_want(q, *clean, table, lens, 0, 0, D ** -0.5, dtype)
    fine = np.ones(got.shape, bool)
    fine[..., 7], fine[2, :, 9] = False, False
    if dtype != "float32":
        tol = tol + P.HALF_STEP[dtype] ** 2 * np.abs(on.from_storage(clean[1], dtype)).max() * 1.05
    P.check(f"shared {dtype} batch {batch}", got[fine], want[fine], tol[fine])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_packed(dtype):
    """A sequence of few rows and one of many."""
    rng = np.random.default_rng(32)
    Hq, Hkv, lens, new = 3, 1, np.array([20, 20]), np.array([2, 60])
    table = P.shuffled_table(rng, lens + new, PAGE, 6, 12)
    kp, vp = (rng.standard_normal((12, Hkv, PAGE, D)).astype(np.float32) for _ in "kv")
    q = P.values(rng, (62, Hq, D), dtype)
    vp[table[:, 0], 0, 3, 7] = np.inf
    k, v = (P.dev(on.to_storage(x, dtype), dtype) for x in (kp, vp))
    got = P.back(paged_attention_packed(P.dev(q, dtype), k, v, P.int32(table), P.int32(lens), P.int32([0, 2, 62]), Hq, Hkv, 60), dtype)
    assert not np.isfinite(got[..., 7]).any() and np.isfinite(np.delete(got, 7, -1)).all()
