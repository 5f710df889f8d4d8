"""Shared-prefix attention rounds no weight to a 16-bit type, however many query rows share a key: its results are as near the 64-bit
form as paged_attention_decode's.

Tolerance: tests/_paged.py's without rounded weights, and for weights in two words the second one's rounding, half a step of half a
step.  Queries are small, so that outputs are far smaller than sum p_j |v_j| and a rounded weight shows."""

import numpy as np
import pytest

from oracle import numerics as on
from oracle import paged as op
from tests import _paged as P

HQ, HKV = 6, 2
CASES = [("float16", 64, 20, 50), ("bfloat16", 64, 20, 50), ("float16", 128, 90, 37), ("bfloat16", 128, 90, 37), ("bfloat16", 64, 45, 130),
         ("bfloat16", 128, 12, 300)]


def made(dtype, D, batch, shared):
    """Sequences of 1 to 40 own positions behind `shared` ones: (lens, table, kp, vp, q)."""
    rng = np.random.default_rng(22)
    lens = shared + rng.integers(1, 41, batch)
    max_pages, n_pages = -(-int(lens.max()) // 16), sum(-(-int(t) // 16) for t in lens) + 2
    table = P.shuffled_table(rng, lens, 16, max_pages, n_pages)
    table[1:, :-(-shared // 16)] = table[0, :-(-shared // 16)]
    kp, vp = (P.values(rng, (n_pages, HKV, 16, D), dtype) for _ in "kv")
    q = on.to_storage((rng.standard_normal((batch, HQ, D)) / 4).astype(np.float32), dtype)
    return lens, table, kp, vp, q


def outputs(made_of, dtype, D):
    """Per sequence and head: (sequence, head, 64-bit output, its tolerance, the output by weights rounded to the type)."""
    lens, table, kp, vp, q = made_of
    kf, vf = (on.from_storage(x, dtype).astype(np.float64) for x in (kp, vp))
    for b, n in enumerate(lens):
        k, _ = op.gather(kf, table[b], n)
        v, _ = op.gather(vf, table[b], n)
        keep = np.ones((1, n), bool)
        for h in range(HQ):
            g = h // (HQ // HKV)
            qh = on.from_storage(q[b, h:h + 1], dtype).astype(np.float64)
            want, weight = op.attend(qh, k[g], v[g], keep, D ** -0.5)
            err = op.score_error(qh, k[g], keep, D ** -0.5, D + 4)
            tol = P.allowed(dtype, want, weight, err, n, False) + P.HALF_STEP[dtype] ** 2 * weight * 1.05
            s = qh @ k[g].T * D ** -0.5
            p = np.exp(s - s.max())
            rounded = on.round_to(p.astype(np.float32), dtype).astype(np.float64) @ v[g] / p.sum()
            yield b, h, want[0], tol[0], rounded[0]


@pytest.mark.parametrize("dtype,D,batch,shared", CASES)
def test_rounded_weights_fall_outside(dtype, D, batch, shared):
    """The oracle with rounded weights, its result not rounded any more."""
    worst = max(float((np.abs(rounded - want) / tol).max()) for _, _, want, tol, rounded in outputs(made(dtype, D, batch, shared), dtype, D))
    assert worst > 2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D,batch,shared", CASES)
def test_many_rows_have_whole_weights(dtype, D, batch, shared):
    from triton_llm.kernels import paged_attention_shared, plan_shared_attention
    lens, table, kp, vp, q = m = made(dtype, D, batch, shared)
    plan = plan_shared_attention(P.int32(table), P.int32(lens), P.int32(np.arange(batch)), P.int32([0, batch]), P.int32([shared]), HQ,
                                 HKV, D, 16, P.H.GPU_DTYPES[dtype])
    got = P.back(paged_attention_shared(P.dev(q, dtype), P.dev(kp, dtype), P.dev(vp, dtype), P.int32(table), plan, HQ, HKV), dtype)
    for b, h, want, tol, _ in outputs(m, dtype, D):
        P.check(f"whole weights {dtype} d{D} sequence {b} head {h}", got[b, h], want, tol)
