"""Weights of packed sequences of at most 32 query rows a KV head are not rounded to a 16-bit type.

Tolerance: tests/_paged.py's without rounded weights, and for weights in two words the second one's rounding, half a step of half a
step.  The inputs have outputs far smaller than sum p_j |v_j|, where a rounded weight shows: a plain form with rounded
weights is shown to fall outside on the CPU."""

import numpy as np
import pytest

from oracle import numerics as on
from oracle import paged as op
from tests import _paged as P

CASES = [("float16", 4, 2, 64, 0, 0), ("bfloat16", 4, 2, 64, 0, 0), ("bfloat16", 4, 2, 128, 0, 0), ("float16", 3, 1, 128, 0, 0),
         ("bfloat16", 16, 1, 64, 20, 3), ("bfloat16", 32, 1, 64, 0, 0)]


def made(dtype, Hq, Hkv, D):
    """Sequences of 1 .. 32 rows a KV head on few keys: (lens, new, starts, table, kp, vp, q)."""
    rng = np.random.default_rng(21)
    G = Hq // Hkv
    new = np.array([m for m in (1, 2, 4, 8, 10, 16, 32) if m * G <= 32] * 3)
    lens = rng.integers(3, 60, new.size)
    total = lens + new
    max_pages, n_pages = -(-int(total.max()) // 16), sum(-(-int(t) // 16) for t in total) + 2
    table = P.shuffled_table(rng, total, 16, max_pages, n_pages)
    kp, vp = (P.values(rng, (n_pages, Hkv, 16, D), dtype) for _ in "kv")
    starts = np.concatenate([[0], np.cumsum(new)])
    q = on.to_storage((rng.standard_normal((int(starts[-1]), Hq, D)) / 4).astype(np.float32), dtype)  # small scores, small errors of them
    return lens, new, starts, table, kp, vp, q


def outputs(made_of, dtype, Hq, Hkv, D, window, sinks):
    """Per sequence and head: (sequence, rows, head, 64-bit output, its tolerance, the output by weights rounded to the type)."""
    lens, new, starts, table, kp, vp, q = made_of
    kf, vf = (on.from_storage(x, dtype).astype(np.float64) for x in (kp, vp))
    for b, (n, m) in enumerate(zip(lens, new)):
        k, _ = op.gather(kf, table[b], n + m)
        v, _ = op.gather(vf, table[b], n + m)
        keep = op.seen(n + np.arange(m), n + m, window, sinks)
        for h in range(Hq):
            g = h // (Hq // Hkv)
            qh = on.from_storage(q[starts[b]:starts[b + 1], h], dtype).astype(np.float64)
            want, weight = op.attend(qh, k[g], v[g], keep, D ** -0.5)
            err = op.score_error(qh, k[g], keep, D ** -0.5, D + 4)
            tol = P.allowed(dtype, want, weight, err, n + m, False) + P.HALF_STEP[dtype] ** 2 * weight * 1.05
            s = np.where(keep, qh @ k[g].T * D ** -0.5, -np.inf)
            p = np.exp(s - s.max(-1, keepdims=True))
            rounded = on.round_to(p.astype(np.float32), dtype).astype(np.float64) @ v[g] / p.sum(-1, keepdims=True)
            yield b, slice(starts[b], starts[b + 1]), h, want, tol, rounded


@pytest.mark.parametrize("dtype,Hq,Hkv,D,window,sinks", CASES)
def test_rounded_weights_fall_outside(dtype, Hq, Hkv, D, window, sinks):
    """The oracle with rounded weights, its result not rounded any more."""
    worst = {}
    for b, _, _, want, tol, rounded in outputs(made(dtype, Hq, Hkv, D), dtype, Hq, Hkv, D, window, sinks):
        worst[b] = max(worst.get(b, 0), float((np.abs(rounded - want) / tol).max()))
    assert max(worst.values()) > 2, worst


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,Hq,Hkv,D,window,sinks", CASES)
def test_few_rows_have_whole_weights(dtype, Hq, Hkv, D, window, sinks):
    from triton_llm.kernels import paged_attention_packed
    lens, new, starts, table, kp, vp, q = m = made(dtype, Hq, Hkv, D)
    got = P.back(paged_attention_packed(P.dev(q, dtype), P.dev(kp, dtype), P.dev(vp, dtype), P.int32(table), P.int32(lens),
                                        P.int32(starts), Hq, Hkv, int(new.max()), window=window, sinks=sinks), dtype)
    for b, at, h, want, tol, _ in outputs(m, dtype, Hq, Hkv, D, window, sinks):
        P.check(f"whole weights {dtype} {Hq}/{Hkv} d{D} sequence {b} head {h}", got[at, h], want, tol)
