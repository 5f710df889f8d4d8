"""Plain 64-bit forms of the paged cache's operators, windowed attention and beam selection.

The reference has none of these; they are written from the operators' definitions
(include/triton_llm_hip.h) and pinned by tests/test_oracle_paged.py.
"""

from __future__ import annotations

import numpy as np

from . import numerics as on


def seen(pos, n_keys: int, window: int = 0, sinks: int = 0) -> np.ndarray:
    """Which of n_keys keys queries at positions pos (rows,) see: (rows, n_keys)."""
    pos = np.asarray(pos, np.int64)[:, None]
    j = np.arange(n_keys)[None]
    keep = j <= pos
    if window > 0:
        keep &= (j > pos - window) | (j < sinks)
    return keep


def attend(q, k, v, keep, scale: float):
    """q (rows, D) over k / v (keys, D), float64: (out, weight) with weight = sum_j p_j |v_j|, what an
    error relative to each p_j or v_j is a fraction of.  Rows without keys give zeros."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    s = np.where(keep, (q @ np.where(keep.any(0)[:, None], k, 0).T) * scale, -np.inf)
    m = s.max(-1, keepdims=True, initial=-np.inf)
    p = np.exp(s - np.where(np.isinf(m), 0, m))
    total = p.sum(-1, keepdims=True)
    p /= np.where(total == 0, 1, total)
    v = np.where(keep.any(0)[:, None], v, 0)
    return p @ v, p @ np.abs(v)


def score_error(q, k, keep, scale: float, n_terms: int) -> np.ndarray:
    """A bound (rows,) on a 32-bit score's error: n_terms roundings of the sum of |q_d k_d|."""
    k = np.where(keep.any(0)[:, None], np.asarray(k, np.float64), 0)
    size = (np.abs(np.asarray(q, np.float64)) @ np.abs(k).T) * abs(scale)
    return np.where(keep, size, 0).max(-1, initial=0) * n_terms * 2.0 ** -24


def gather(pages, row, n: int):
    """(values (n_kv, n, D) float64, there (n,)) of the first n positions; pages that are not there read as 0."""
    n_pages, n_kv, ps, D = pages.shape
    out = np.zeros((n_kv, n, D))
    there = np.zeros(n, bool)
    for t in range(n):
        p = int(row[t // ps])
        if 0 <= p < n_pages:
            out[:, t] = pages[p, :, t % ps]
            there[t] = True
    return out, there


def rotate(x, c, s, interleaved: bool):
    """x (..., d) float32, c / s (..., r / 2): the first r features turned, products and sums rounded one by one."""
    x = np.array(x, np.float32)
    half = c.shape[-1]
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    xa, xb = x[..., a].copy(), x[..., b].copy()
    x[..., a] = xa * c - xb * s
    x[..., b] = xa * s + xb * c
    return x


def append(q, k_new, v_new, k_pages, v_pages, table, lens, cos=None, sin=None, new_lens=None, q_out=None,
           interleaved=False, dtype="float32"):
    """Storage arrays in, (q_out, k_pages, v_pages) copies out, bit for bit.  q_out: what is there before."""
    n_pages, _, ps, _ = k_pages.shape
    kp, vp = k_pages.copy(), v_pages.copy()
    qo = None if q is None else (q if q_out is None else q_out).copy()
    B, n = k_new.shape[:2]
    for b in range(B):
        for t in range(n if new_lens is None else min(n, int(new_lens[b]))):
            pos = int(lens[b]) + t
            if pos < 0 or pos >= table.shape[1] * ps or (cos is not None and pos >= cos.shape[0]):
                continue
            page = int(table[b, pos // ps])
            if not 0 <= page < n_pages:
                continue

            def turn(x):
                if cos is None:
                    return x
                return on.to_storage(on.round_to(rotate(on.from_storage(x, dtype), cos[pos], sin[pos], interleaved),
                                                 dtype), dtype)

            kp[page, :, pos % ps] = turn(k_new[b, t])
            vp[page, :, pos % ps] = v_new[b, t]
            if q is not None:
                qo[b, t] = turn(q[b, t])
    return qo, kp, vp


def beam_select(logits, scores, n: int):
    """logits (batch, beams, vocab), scores (batch, beams): (scores, parents, tokens), (batch, n) each."""
    B, J, V = logits.shape
    x = np.asarray(logits, np.float64)
    out_s, out_p, out_t = np.full((B, n), -np.inf), np.full((B, n), -1, np.int32), np.full((B, n), -1, np.int32)
    for b in range(B):
        total = np.full((J, V), -np.inf)
        for j in range(J):
            m = x[b, j].max()
            if not (np.isfinite(m) and np.isfinite(scores[b, j])) or np.isnan(x[b, j]).any():
                continue
            total[j] = np.float64(scores[b, j]) + (x[b, j] - (m + np.log(np.exp(x[b, j] - m).sum())))
        flat = total.ravel()
        at = np.argsort(-flat, kind="stable")[:n]
        at = at[flat[at] > -np.inf]
        out_s[b, :at.size], out_p[b, :at.size], out_t[b, :at.size] = flat[at], at // V, at % V
    return out_s, out_p, out_t
