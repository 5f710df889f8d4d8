"""What the paged cache's GPU tests share: pools behind shuffled page tables, and how far an attention
output may be from the 64-bit one."""

from __future__ import annotations

import numpy as np

from oracle import numerics as on
from oracle import paged as op
from tests import _helpers as H
from triton_llm import gpu

HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def values(rng, shape, dtype):
    """Normal values as storage."""
    return on.to_storage(rng.standard_normal(shape).astype(np.float32), dtype)


def shuffled_table(rng, lens, page, max_pages, n_pages, spare=-1):
    """(batch, max_pages) int32: the pages of lens[b] positions anywhere in the pool, `spare` behind them."""
    order = iter(rng.permutation(n_pages))
    table = np.full((len(lens), max_pages), spare, np.int32)
    for b, n in enumerate(lens):
        for i in range(min(max_pages, -(-max(int(n), 0) // page))):
            table[b, i] = next(order)
    return table


def pool_with(rng, table, keep, shape, dtype):
    """A pool (n_pages, n_kv, page, D) that holds NaN but where keep[b] (positions,) names positions of sequence b."""
    pool = np.full(shape, on.nan_storage(dtype), on.storage_dtype(dtype))
    page = shape[2]
    for b, k in enumerate(keep):
        for t in np.flatnonzero(k):
            p = int(table[b, t // page])
            if 0 <= p < shape[0]:
                pool[p, :, t % page] = values(rng, (shape[1], shape[3]), dtype)
    return pool


def allowed(dtype, out, weight, score_err, n_keys, rounded_weights):
    """How far an output may be from the 64-bit `out` (rows, D).

    With p_j the weights, sum p_j = 1, and W = sum p_j |v_j|: a relative error r of every exp(s_j) changes
    out by at most 2 r W (once in the sum over v, once in the sum of weights).  r is the score's
    own error (score_err), that of the exponent's product and subtraction in log2 units, of the order of
    the exponents left (|s - m| <= 60 counts: below that p_j < 2^-60), 60 * 2^-23, and the hardware exp2's, 2^-22.  Weights rounded to
    16 bits add half a step each, once.  Sums of n_keys terms with rescaling add n_keys + 64 roundings
    of 2^-24 in either sum, and the result is rounded once."""
    r = score_err[:, None] + 60 * 2.0 ** -23 + 2.0 ** -22
    sums = 2 * (n_keys + 64) * 2.0 ** -24
    weights = HALF_STEP[dtype] if rounded_weights else 0.0
    tiny = 2.0 ** -24 if dtype == "float16" else 0.0  # fp16's smallest step
    return (2 * r + sums + weights) * weight * 1.05 + HALF_STEP[dtype] * np.abs(out) * 1.05 + tiny + 1e-30


def check(name, got, want, tol):
    assert np.isfinite(got).all(), f"{name}: not finite"
    worst = float((np.abs(got - want) / tol).max(initial=0))
    print(f"[{'PASS' if worst <= 1 else 'FAIL'}] {name}: {worst:.3f} of what is allowed", flush=True)
    assert worst <= 1, f"{name}: {worst} of what is allowed"


def dev(x, dtype):
    return H.upload(x, dtype)


def back(t, dtype):
    return on.from_storage(H.download(t), dtype)


def int32(x):
    return gpu.to_device(np.ascontiguousarray(x, np.int32))


def decode_want(q, kp, vp, table, lens, window, sinks, scale, dtype):
    """(want, allowed) of one query per sequence (batch, H, D), from storage arrays."""
    B, Hq, D = q.shape
    Hkv = kp.shape[1]
    cap = table.shape[1] * kp.shape[2]
    kf, vf = on.from_storage(kp, dtype), on.from_storage(vp, dtype)
    want, tol = np.zeros((B, Hq, D)), np.full((B, Hq, D), 1e-30)
    for b in range(B):
        n = min(max(int(lens[b]), 0), cap)
        if n == 0:
            continue
        k, there = op.gather(kf, table[b], n)
        v, _ = op.gather(vf, table[b], n)
        keep = op.seen([n - 1], n, window, sinks) & there
        for h in range(Hq):
            qh = on.from_storage(q[b, h:h + 1], dtype)
            o, w = op.attend(qh, k[h // (Hq // Hkv)], v[h // (Hq // Hkv)], keep, scale)
            e = op.score_error(qh, k[h // (Hq // Hkv)], keep, scale, D + 4)
            want[b, h], tol[b, h] = o[0], allowed(dtype, o, w, e, n, False)[0]
    return want, tol


def rows_want(q, k, v, pos, keep_extra, window, sinks, scale, dtype):
    """(want, allowed) of rows q (H, rows, D) at positions pos over k / v (Hkv, keys, D) float64."""
    Hq, _, D = q.shape
    Hkv, n, _ = k.shape
    keep = op.seen(pos, n, window, sinks) & keep_extra
    want, tol = np.zeros(q.shape), np.zeros(q.shape)
    for h in range(Hq):
        qh = on.from_storage(q[h], dtype)
        o, w = op.attend(qh, k[h // (Hq // Hkv)], v[h // (Hq // Hkv)], keep, scale)
        e = op.score_error(qh, k[h // (Hq // Hkv)], keep, scale, D + 4)
        want[h], tol[h] = o, allowed(dtype, o, w, e, n, dtype != "float32")
    return want, tol
