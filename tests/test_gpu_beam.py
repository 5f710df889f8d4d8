"""Beam search's selection on the GPU against the 64-bit form: parents and tokens exactly, scores to half a
32-bit step and the error of the log-sum-exp (every exp within 2^-22 of its value, hence their sum, hence
its logarithm by as much)."""

import numpy as np
import pytest

from oracle import numerics as on
from oracle import paged as op
from tests import _paged as P
from triton_llm import gpu
from triton_llm.kernels import beam_select

pytestmark = pytest.mark.gpu


def run(logits, scores, n, dtype="float32"):
    B, J = scores.shape
    x = on.to_storage(logits, dtype)
    out = beam_select(P.dev(x, dtype), gpu.to_device(np.asarray(scores, np.float32)), n)
    got = [gpu.to_host(t) for t in out]
    want = op.beam_select(on.from_storage(x, dtype).reshape(B, J, -1), np.asarray(scores, np.float32), n)
    np.testing.assert_array_equal(got[1], want[1], err_msg="parents")
    np.testing.assert_array_equal(got[2], want[2], err_msg="tokens")
    fine = np.isfinite(want[0])
    np.testing.assert_array_equal(np.isfinite(got[0]), fine)
    assert (got[0][~fine] == -np.inf).all()
    np.testing.assert_allclose(got[0][fine], want[0][fine], rtol=1.01 * 2.0 ** -24, atol=2.0 ** -22)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("B,J,V,n", [(1, 4, 50257, 8), (3, 5, 1000, 10), (2, 1, 1, 1), (1, 2, 1, 4), (1, 1, 63, 64), (2, 3, 65, 7),
                                     (1, 64, 300, 64), (5, 7, 2049, 14), (1, 8, 128256, 16), (40, 2, 500, 3),
                                     (1, 8, 128256, 20), (2, 16, 20000, 64), (1, 2, 262144, 33)])
def test_normal_logits(dtype, B, J, V, n):
    rng = np.random.default_rng(V)
    run(2.5 * rng.standard_normal((B * J, V)), -rng.uniform(3, 9, (B, J)), n, dtype)


def test_ties_go_to_the_lowest_place():
    run(np.zeros((4, 5000)), np.zeros((1, 4)), 64)                       # everything equal
    run(np.zeros((4, 5000)), np.array([[-2, -1, -1, -3.0]]), 9)
    run(np.zeros((8, 20000)), np.zeros((1, 8)), 12)
    run(np.zeros((8, 20000)), np.zeros((1, 8)), 40)
    x = np.zeros((2, 9000))
    x[:, 4000:8000] = 5
    run(x, np.zeros((1, 2)), 40)
    run(np.repeat(np.arange(100.0), 90)[None] / 10, np.zeros((1, 1)), 64, "bfloat16")


@pytest.mark.parametrize("order", [1, -1])
@pytest.mark.parametrize("n", [1, 16, 64])
def test_rows_in_order(order, n):
    x = np.linspace(-20, 20, 30000)[::order]
    run(np.stack([x, x + 0.001, x[::-1]]), np.array([[-1.0, -1.5, -1.2]]), n)


def test_clustered_rows():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((3, 40000))
    x[0, 640:3000] += 30  # the best all lie in neighbouring groups
    x[1, 12345] = 50
    run(x, np.array([[-3.0, -3.1, -2.9]]), 64)


def test_masked_and_undefined_rows():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((8, 3000))
    x[0] = -np.inf
    x[1, 5] = np.nan
    x[2, 7] = np.inf
    x[3, 3:] = -np.inf
    x[4, ::2] = -np.inf
    x[7] = np.nan
    scores = np.array([[-1, -1, -1, -2.0], [-1, -np.inf, np.nan, -1]])
    run(x, scores, 40)
    run(x[:4], scores[:1], 20)   # three continuations for twenty places
    run(x[:4, :2], np.full((1, 4), -np.inf), 6)
    y = rng.standard_normal((2, 3000))
    y[:, 100:200] = np.finfo(np.float32).min  # masks of the type's lowest value
    run(y, np.zeros((1, 2)), 64)
    y[:, 3:] = np.finfo(np.float32).min
    run(y, np.zeros((1, 2)), 8)


def test_far_apart_scores_and_large_logits():
    rng = np.random.default_rng(2)
    run(1e4 * rng.standard_normal((4, 5000)), np.array([[-1e5, 0, -1e30, -3e4]]), 12)


def test_captured_call_replays():
    rng = np.random.default_rng(3)
    x = gpu.to_device(rng.standard_normal((8, 5000)).astype(np.float32))
    s = gpu.to_device(-rng.uniform(1, 3, (2, 4)).astype(np.float32))
    want = [gpu.to_host(t) for t in beam_select(x, s, 8)]
    out = tuple(gpu.zeros((2, 8), t) for t in (np.float32, np.int32, np.int32))
    gpu.synchronize()
    with gpu.capture() as g:
        beam_select(x, s, 8, out=out)
    for _ in range(3):
        for t in out:
            t.from_numpy(np.zeros((2, 8), t.dtype))
        beam_select(x, s, 3)  # eager work on the shared workspace
        g.replay()
        for t, w in zip(out, want):
            np.testing.assert_array_equal(gpu.to_host(t), w)
