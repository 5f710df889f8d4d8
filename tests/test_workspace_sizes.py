"""What a caller asks for a workspace's size is what the calls ask of the workspace."""

import ctypes

import numpy as np
import pytest

from triton_llm import gpu
from triton_llm.kernels import (beam_select, beam_workspace_bytes, paged_attention_prefill, paged_prefill_workspace_bytes,
                                window_attention, window_workspace_bytes)
from triton_llm.kernels import _common


def fake(shape, dtype=np.float32, nbytes=0):
    return gpu.DeviceTensor(ctypes.c_void_p(None), shape, dtype, nbytes, defer_free=False)


def calls():
    bf = gpu.bfloat16
    q, k = fake((1, 12, 300, 128), bf), fake((1, 4, 5000, 128), bf)
    pool, i32 = fake((900, 4, 16, 64), np.float16), lambda *s: fake(s, np.int32)
    rows = fake((8, 500, 12, 64), np.float16)
    paged = (rows, pool, pool, i32(8, 300), i32(8), 12, 4)
    counts = [0, 500, 0, 0, 1, 0, 0, 0]
    x, s = fake((32, 5000)), fake((4, 8))
    out = (fake((4, 16)), i32(4, 16), i32(4, 16))
    return [
        ("window", window_workspace_bytes(1, 12, 4, 300, 5000, 128, bf), lambda ws: window_attention(q, k, k, 0, out=q, workspace=ws)),
        ("window 700", window_workspace_bytes(1, 12, 4, 300, 5000, 128, bf, 700, 4),
         lambda ws: window_attention(q, k, k, 700, 4, out=q, workspace=ws)),
        ("paged", paged_prefill_workspace_bytes(8, 12, 4, 500, 4800, 64, np.float16),
         lambda ws: paged_attention_prefill(*paged, new_lens=i32(8), out=rows, workspace=ws)),
        ("paged, counted", paged_prefill_workspace_bytes(8, 12, 4, 500, 4800, 64, np.float16, host_new_lens=counts),
         lambda ws: paged_attention_prefill(*paged, new_lens=i32(8), out=rows, workspace=ws, host_new_lens=counts)),
        ("beam", beam_workspace_bytes(4, 8, 5000), lambda ws: beam_select(x, s, 16, out=out, workspace=ws)),
    ]


@pytest.mark.parametrize("i", range(5))
def test_size_is_what_a_call_asks(monkeypatch, i):
    asked = []
    monkeypatch.setattr(gpu, "runtime", lambda: type("R", (), {"__getattr__": lambda s, n: lambda *a: asked.append(n) or 0})())
    name, need, call = calls()[i]
    assert need > 0, name
    call(fake((need,), np.uint8, need))
    assert len(asked) == 1
    with pytest.raises(ValueError, match=f"{need} required"):
        call(fake((need - 1,), np.uint8, need - 1))
    assert _common._recording is None


def test_sizes_refuse():
    with pytest.raises(ValueError, match="multiple"):
        paged_prefill_workspace_bytes(1, 5, 2, 10, 64, 64, np.float32)
    with pytest.raises(ValueError, match="multiple"):
        paged_prefill_workspace_bytes(1, 4, 0, 10, 64, 64, np.float32)
    with pytest.raises(ValueError, match="must hold 2"):
        paged_prefill_workspace_bytes(2, 4, 2, 10, 64, 64, np.float32, host_new_lens=[1])
    with pytest.raises(ValueError, match="window and sinks"):
        window_workspace_bytes(1, 4, 2, 10, 64, 64, np.float32, window=-1)
    assert beam_workspace_bytes(1, 65, 100) == 0 and window_workspace_bytes(1, 4, 2, 4, 16, 64, np.float32) == 0
