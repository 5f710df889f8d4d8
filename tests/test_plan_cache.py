"""What the wrappers keep of a call's shapes does not outlive the device limits that it was planned under."""

import ctypes

import numpy as np
import pytest

from tests import _paged as P
from triton_llm import _lib, gpu
from triton_llm.kernels import paged, paged_attention_prefill, window, window_attention


def test_kept_plans_are_forgotten(monkeypatch):
    class Runtime:
        def tl_init(self, device):
            return 0

    def plans():
        s = (64, 64, 64)
        pool, lens = (9, 2, 16, 64), (3,)
        return (window._strided_plan(1, 4, 2, 8, 900, 64, s, s, s, s, 0, 0),
                paged._attention_plan(pool, pool, (3, 70), lens, None, (3, 6, 4, 64), 4, 2, 0, 0, True))

    monkeypatch.setattr(gpu, "_rt", Runtime())
    monkeypatch.setattr(gpu, "_initialized", True)
    first = plans()
    assert [a is b for a, b in zip(plans(), first)] == [True, True]
    gpu.reload_overrides()
    assert [a is b for a, b in zip(plans(), first)] == [False, False]


@pytest.mark.gpu
def test_calls_after_a_limit_is_lifted(monkeypatch):
    """The same bits, divided keys among them, as without the limit before."""
    rng = np.random.default_rng(0)
    q, k, v = (P.dev(P.values(rng, s, "float32"), "float32") for s in [(1, 4, 100, 64), (1, 2, 900, 64), (1, 2, 900, 64)])
    pool = [gpu.DeviceTensor(ctypes.c_void_p(t.data_ptr()), (112, 1, 16, 64), t.dtype, t.nbytes, defer_free=False) for t in (k, v)]
    table, lens = P.int32(np.arange(112).reshape(2, 56)), P.int32([796, 700])
    rows = gpu.view(q, (2, 50, 4, 64))

    def calls():
        return [gpu.to_host(window_attention(q, k, v, 0)),
                gpu.to_host(paged_attention_prefill(rows, *pool, table, lens, 4, 1))]

    want = calls()
    P.H.set_override(monkeypatch, "TRITON_LLM_HIP_MAX_CUS", 1)
    limited = calls()
    P.H.set_override(monkeypatch, "TRITON_LLM_HIP_MAX_CUS", None)
    for a, b, c in zip(calls(), want, limited):
        np.testing.assert_array_equal(a, b)
        assert (a != c).any()  # the limit takes another path


@pytest.mark.gpu
def test_calls_planned_under_a_limit(monkeypatch):
    """Shapes that the limit sees first are divided once it is lifted, as the same shapes under another name are."""
    rng = np.random.default_rng(1)
    q, k, v = (P.dev(P.values(rng, s, "float32"), "float32") for s in [(1, 4, 90, 64), (1, 2, 1100, 64), (1, 2, 1100, 64)])
    P.H.set_override(monkeypatch, "TRITON_LLM_HIP_MAX_CUS", 1)
    limited = gpu.to_host(window_attention(q, k, v, 0))
    P.H.set_override(monkeypatch, "TRITON_LLM_HIP_MAX_CUS", None)
    want = gpu.to_host(window_attention(q, k, v, 1 << 30))  # a window that hides nothing
    np.testing.assert_array_equal(gpu.to_host(window_attention(q, k, v, 0)), want)
    assert (limited != want).any()
    assert _lib.load().tl_window_workspace_bytes(1, 4, 2, 90, 1100, 64, 0, 0, _lib.DTYPE_F32) > 0
