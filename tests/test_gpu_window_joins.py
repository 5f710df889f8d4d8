"""Divided keys: how many parts a row tile has, by the deal's own arithmetic, and that parts joined by the waves and by a
second launch give the same."""

import numpy as np
import pytest

from oracle import numerics as on
from tests import _paged as P
from triton_llm import gpu
from triton_llm.kernels import window_attention

pytestmark = pytest.mark.gpu
ROWS, LEAST, WAVE_PARTS = 128, 4, 4  # rows of a tile, key tiles of a part at least, parts that the waves join


def slots_of(cus, dtype, D):
    return cus * (2 if D == 128 else 1 if dtype == "float32" else 3)


def parts_of(Sq, Sk, Hq, Hkv, D, dtype, cus):
    """(parts of a row tile, whether the waves join them) of one causal sequence whose keys are divided."""
    bn, slots = 32 if dtype == "float32" else 64, slots_of(cus, dtype, D)
    tiles, keys = -(-Sq * (Hq // Hkv) // ROWS), -(-Sk // bn)
    assert tiles * Hkv < slots and keys >= 2 * LEAST  # else undivided
    aim = max(slots - tiles * Hkv, slots // 2)
    share = max(int(tiles * keys * Hkv / aim * 1.00001) + 1, LEAST)
    return -(-keys // share), slots <= WAVE_PARTS * tiles * Hkv


def make(dtype, D, Hq, Hkv, Sq, Sk, seed=11):
    rng = np.random.default_rng(seed)
    return [P.values(rng, s, dtype) for s in [(1, Hq, Sq, D), (1, Hkv, Sk, D), (1, Hkv, Sk, D)]]


def check(name, got, x, dtype):
    q, k, v = x
    Sq, Sk, D = q.shape[2], k.shape[2], q.shape[3]
    want, tol = P.rows_want(q[0], on.from_storage(k[0], dtype), on.from_storage(v[0], dtype), Sk - Sq + np.arange(Sq), True, 0, 0,
                            D ** -0.5, dtype)
    P.check(name, got[0], want, tol)


@pytest.mark.parametrize("dtype,D,cus", [("float32", 64, 24), ("float32", 128, 12), ("float16", 64, 8), ("float16", 128, 12),
                                         ("bfloat16", 128, 10), ("bfloat16", 64, 9)])
def test_waves_join_two_parts_and_more(monkeypatch, dtype, D, cus):
    """From a workspace that holds anything, eager and replayed with other calls on the same workspace between, always
    the same bits."""
    P.H.set_override(monkeypatch, "TRITON_LLM_HIP_MAX_CUS", cus)
    Hq, Hkv, Sq, Sk = 4, 2, 200, 600
    parts, by_waves = parts_of(Sq, Sk, Hq, Hkv, D, dtype, cus)
    assert parts >= 2 and by_waves, (parts, by_waves)
    x = make(dtype, D, Hq, Hkv, Sq, Sk)
    on_dev = [P.dev(t, dtype) for t in x]
    others = [P.dev(t, dtype) for t in make(dtype, D, Hq, Hkv, 150, 700, 12)]
    ws = gpu.to_device(np.full(1 << 24, 0xFF, np.uint8))
    first = P.back(window_attention(*on_dev, 0, workspace=ws), dtype)
    check(f"{parts} parts {dtype} d{D}", first, x, dtype)
    out = P.dev(np.zeros(x[0].shape, x[0].dtype), dtype)
    gpu.synchronize()
    with gpu.capture() as g:
        window_attention(*on_dev, 0, out=out, workspace=ws)
    for i in range(4):
        out.from_numpy(np.full(x[0].shape, on.nan_storage(dtype), x[0].dtype))
        if i % 2:
            window_attention(*others, 0, workspace=ws)
        g.replay()
        np.testing.assert_array_equal(P.back(out, dtype), first)
        np.testing.assert_array_equal(P.back(window_attention(*on_dev, 0, workspace=ws), dtype), first)


@pytest.mark.parametrize("dtype,D,cus", [("float32", 64, 40), ("float32", 128, 30), ("float16", 64, 20), ("bfloat16", 128, 40)])
def test_second_launch_joins_many_parts(monkeypatch, dtype, D, cus):
    P.H.set_override(monkeypatch, "TRITON_LLM_HIP_MAX_CUS", cus)
    Hq, Hkv, Sq, Sk = 4, 2, 100, 2000
    parts, by_waves = parts_of(Sq, Sk, Hq, Hkv, D, dtype, cus)
    assert parts > 4 and not by_waves, (parts, by_waves)
    x = make(dtype, D, Hq, Hkv, Sq, Sk)
    check(f"{parts} parts {dtype} d{D}", P.back(window_attention(*(P.dev(t, dtype) for t in x), 0), dtype), x, dtype)
