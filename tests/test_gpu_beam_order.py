"""Continuations of different beams whose scores differ by far less than a 32-bit step of the log-sum-exp: the order is that
of the 64-bit scores."""

import numpy as np
import pytest

from oracle import numerics as on
from oracle import paged as op
from tests import _paged as P
from triton_llm import gpu
from triton_llm.kernels import beam_select

pytestmark = pytest.mark.gpu


def log_sum_exp(x):
    m = x.max()
    return m + np.log(np.exp(x - m).sum())


def level_beams(rng, J, V, dtype, spread):
    """(logits (J, V) as stored values, scores (1, J) float32): one high entry a row over a floor that is the same everywhere in
    the row, or in two thirds of it, and another in every row; scores chosen so that the rows' best continuations agree
    to a float32 step of the scores."""
    x = np.repeat(-8 - rng.permutation(64)[:J, None] / 16, V, axis=1)
    for row in x:
        some = rng.choice(V, V // 3, replace=False)
        row[some] += spread * rng.standard_normal(some.size)
        row[rng.integers(V)] = 0
    x = on.from_storage(on.to_storage(x.astype(np.float32), dtype), dtype).astype(np.float64)
    top = np.array([r.max() - log_sum_exp(r) for r in x])
    return x, (top.min() - top).astype(np.float32)[None]


@pytest.mark.parametrize("spread", [0.0, 1.0])
@pytest.mark.parametrize("dtype,J,V", [("float32", 8, 128256), ("float32", 4, 50257), ("float32", 16, 2000), ("float16", 6, 30000),
                                       ("bfloat16", 12, 128256)])
def test_order_of_beams_that_are_level(dtype, J, V, spread):
    rng = np.random.default_rng(J + V)
    for _ in range(4):
        x, scores = level_beams(rng, J, V, dtype, spread)
        want = op.beam_select(x[None], scores, J)
        gaps = -np.diff(want[0][0])
        got = [gpu.to_host(t) for t in beam_select(P.dev(on.to_storage(x.astype(np.float32), dtype), dtype),
                                                   gpu.to_device(scores), J)]
        print(f"smallest gap {gaps.min():.2e}, gaps below 2e-7: {(gaps < 2e-7).sum()} of {gaps.size}", flush=True)
        assert gaps.min() > 1e-12  # the 64-bit form itself is not much better
        np.testing.assert_array_equal(got[1], want[1])
        np.testing.assert_array_equal(got[2], want[2])


def test_rows_that_are_one_another_but_for_a_small_entry():
    """Equal scores and rows but for one entry far below: by its mass alone the rows differ, 1e-9 and less."""
    V, far = 40000, np.array([-12.0, -15.0, -18.0, -13.0, -21.0, -16.0], np.float32)
    x = np.full((far.size, V), -9.1, np.float32)
    x[:, 17] = 2.5
    x[np.arange(far.size), 5] = far
    want = op.beam_select(x[None].astype(np.float64), np.zeros((1, far.size)), far.size)
    assert want[1][0].tolist() == np.argsort(far, kind="stable").tolist()
    got = [gpu.to_host(t) for t in beam_select(gpu.to_device(x), gpu.zeros((1, far.size)), far.size)]
    np.testing.assert_array_equal(got[1], want[1])
    np.testing.assert_array_equal(got[2], want[2])
