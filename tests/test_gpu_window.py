"""Attention through a sliding window with sinks on the GPU against the 64-bit form."""

import ctypes

import numpy as np
import pytest

from oracle import numerics as on
from tests import _paged as P
from triton_llm import gpu
from triton_llm.kernels import flash_attention, window_attention, window_attention_strided

pytestmark = pytest.mark.gpu
DTYPES = ["float32", "float16", "bfloat16"]


def run(dtype, B, Hq, Hkv, Sq, Sk, D, window, sinks, scale=None, seed=0):
    rng = np.random.default_rng(seed + Sq + Sk)
    q = P.values(rng, (B, Hq, Sq, D), dtype)
    k, v = P.values(rng, (B, Hkv, Sk, D), dtype), P.values(rng, (B, Hkv, Sk, D), dtype)
    out = P.dev(np.full(q.shape, on.nan_storage(dtype), on.storage_dtype(dtype)), dtype)
    window_attention(P.dev(q, dtype), P.dev(k, dtype), P.dev(v, dtype), window, sinks, sm_scale=scale, out=out)
    got = P.back(out, dtype)
    for b in range(B):
        want, tol = P.rows_want(q[b], on.from_storage(k[b], dtype), on.from_storage(v[b], dtype), Sk - Sq + np.arange(Sq), True,
                                window, sinks, D ** -0.5 if scale is None else scale, dtype)
        P.check(f"window {dtype} {Hq}/{Hkv} {Sq}x{Sk} d{D} window {window} sinks {sinks}", got[b], want, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq,Sk,window,sinks", [(1, 1, 1, 0), (1, 300, 40, 4), (130, 130, 1, 0), (300, 300, 64, 4), (300, 300, 65, 0),
                                                (257, 400, 100, 130), (140, 100, 30, 2), (50, 20, 0, 0), (200, 200, 0, 0),
                                                (200, 200, 1 << 30, 3), (520, 520, 33, 1), (129, 640, 20, 65)])
def test_window(dtype, D, Sq, Sk, window, sinks):
    run(dtype, 1, 2, 1, Sq, Sk, D, window, sinks)


@pytest.mark.parametrize("B,Hq,Hkv", [(2, 6, 2), (3, 5, 5), (1, 9, 3), (1, 8, 1), (1, 40, 1), (1, 160, 1)])
def test_heads_and_batches(B, Hq, Hkv):
    run("bfloat16", B, Hq, Hkv, 200, 210, 64, 50, 3)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 5.0])
def test_scales(scale):
    run("float16", 1, 2, 1, 100, 100, 64, 30, 2, scale=scale)
    run("float32", 1, 2, 1, 100, 100, 64, 0, 0, scale=scale)


@pytest.mark.parametrize("window", [(1 << 31) - 1, 3 << 29, (3 << 29) - 1, 1 << 30])
def test_windows_beyond_every_key(window):
    run("float32", 1, 2, 1, 90, 50, 64, window, 3)  # the first 40 rows stand before position 0
    run("float16", 1, 2, 1, 50, 90, 128, window, 0)


def test_long():
    run("bfloat16", 1, 1, 1, 4000, 4000, 128, 700, 4)


def test_no_window_agrees_with_flash():
    """window = 0 is the causal prefill: both within their rounding of each other."""
    rng = np.random.default_rng(4)
    x = [P.dev(P.values(rng, s, "float32"), "float32") for s in [(1, 4, 300, 64), (1, 2, 300, 64), (1, 2, 300, 64)]]
    a, b = gpu.to_host(window_attention(*x, 0)), gpu.to_host(flash_attention(*x))
    np.testing.assert_allclose(a, b, atol=1e-4)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_rows_in_place(dtype):
    """The projection's (seq, heads * d_k) rows, K and V beside each other, one row apart by more than its size."""
    rng = np.random.default_rng(6)
    S, Hq, Hkv, D = 150, 4, 2, 64
    row = (Hq + 2 * Hkv) * D + 32
    qkv = P.values(rng, (S, row), dtype)
    buf = P.dev(qkv, dtype)
    e = qkv.dtype.itemsize

    def part(first):
        return gpu.DeviceTensor(ctypes.c_void_p(buf.data_ptr() + first * e), (1,), buf.dtype, e, defer_free=False)

    out = P.dev(np.zeros((S, Hq * D + 3), qkv.dtype), dtype)
    window_attention_strided(part(0), part(Hq * D), part((Hq + Hkv) * D), out, batch=1, n_head=Hq, n_kv_head=Hkv, seq_q=S,
                             seq_k=S, d_k=D, q_strides=(0, D, row), k_strides=(0, D, row), v_strides=(0, D, row),
                             o_strides=(0, D, Hq * D + 3), window=40, sinks=2)
    f = on.from_storage(qkv, dtype)
    heads = lambda lo, n: f[:, lo * D:(lo + n) * D].reshape(S, n, D).transpose(1, 0, 2)  # noqa: E731
    qs = qkv[:, :Hq * D].reshape(S, Hq, D).transpose(1, 0, 2)
    want, tol = P.rows_want(np.ascontiguousarray(qs), heads(Hq, Hkv), heads(Hq + Hkv, Hkv), np.arange(S), True, 40, 2, D ** -0.5, dtype)
    got = P.back(out, dtype)
    P.check(f"strided {dtype}", got[:, :Hq * D].reshape(S, Hq, D).transpose(1, 0, 2), want, tol)
    assert (got[:, Hq * D:] == 0).all()


def test_captured_calls_replay():
    rng = np.random.default_rng(2)
    x = [P.dev(P.values(rng, s, "bfloat16"), "bfloat16") for s in [(1, 4, 300, 64), (1, 2, 300, 64), (1, 2, 300, 64)]]
    out = gpu.zeros((1, 4, 300, 64), gpu.bfloat16)
    want = gpu.to_host(window_attention(*x, 100, 4))
    with gpu.capture() as g:
        window_attention(*x, 100, 4, out=out)
    for _ in range(3):
        out.from_numpy(np.zeros((1, 4, 300, 64), np.uint16))
        g.replay()
        window_attention(*x, 50, 0)
        np.testing.assert_array_equal(gpu.to_host(out).view(np.uint16), want.view(np.uint16))


@pytest.mark.parametrize("dtype,D,cus", [("float32", 64, 16), ("float16", 64, 8), ("bfloat16", 128, 10)])
def test_few_parts_joined_without_a_second_launch(monkeypatch, dtype, D, cus):
    """Row tiles of two or three parts: from a workspace that holds anything, eager and replayed with other calls on the
    same workspace between, always the same bits."""
    P.H.set_override(monkeypatch, "TRITON_LLM_HIP_MAX_CUS", cus)
    rng = np.random.default_rng(11)
    B, Hq, Hkv, Sq, Sk = 1, 4, 2, 200, 600
    q, k, v = (P.values(rng, s, dtype) for s in [(B, Hq, Sq, D), (B, Hkv, Sk, D), (B, Hkv, Sk, D)])
    x = [P.dev(t, dtype) for t in (q, k, v)]
    y = [P.dev(P.values(rng, s, dtype), dtype) for s in [(B, Hq, 150, D), (B, Hkv, 700, D), (B, Hkv, 700, D)]]
    ws = gpu.to_device(np.full(1 << 24, 0xFF, np.uint8))
    first = P.back(window_attention(*x, 0, workspace=ws), dtype)
    want, tol = P.rows_want(q[0], on.from_storage(k[0], dtype), on.from_storage(v[0], dtype), Sk - Sq + np.arange(Sq), True, 0, 0,
                            D ** -0.5, dtype)
    P.check(f"few parts {dtype} d{D}", first[0], want, tol)
    out = P.dev(np.zeros(q.shape, q.dtype), dtype)
    gpu.synchronize()
    with gpu.capture() as g:
        window_attention(*x, 0, out=out, workspace=ws)
    for i in range(4):
        out.from_numpy(np.full(q.shape, on.nan_storage(dtype), q.dtype))
        if i % 2:
            window_attention(*y, 0, workspace=ws)
        g.replay()
        np.testing.assert_array_equal(P.back(out, dtype), first)
        np.testing.assert_array_equal(P.back(window_attention(*x, 0, workspace=ws), dtype), first)
