"""plan_shared_attention's len_add is a 32-bit number: others are refused, before any device work."""

import ctypes

import numpy as np
import pytest

from triton_llm import gpu
from triton_llm.kernels import plan_shared_attention


def i32(*shape):
    return gpu.DeviceTensor(ctypes.c_void_p(None), shape, np.int32, 0, defer_free=False)


@pytest.mark.parametrize("len_add", [1 << 31, -(1 << 31) - 1, 1 << 32])
def test_len_add_past_32_bits(len_add):
    with pytest.raises(ValueError, match="len_add"):
        plan_shared_attention(i32(3, 7), i32(3), i32(3), i32(2), i32(1), 4, 2, 64, 16, np.float32, len_add=len_add)
