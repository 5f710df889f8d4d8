"""Outputs that lie over an attention call's inputs are refused; rows side by side in one buffer are not."""

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

from oracle import numerics as on
from tests import _paged as P
from triton_llm import _lib, gpu
from triton_llm.kernels import paged_attention_decode, window_attention, window_attention_strided

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

MAIN = r"""
#include "tl_paged.h"
#include <cstdio>
int main() {  // two tensors a line: base n0 n1 n2 s0 s1 s2 row
  long long v[16];
  while (true) {
    tlpg::Rows3 t[2];
    for (int i = 0; i < 16; ++i)
      if (scanf("%lld", &v[i]) != 1) return 0;
    for (int k = 0; k < 2; ++k)
      t[k] = tlpg::Rows3{(const void*)v[8 * k], {v[8 * k + 1], v[8 * k + 2], v[8 * k + 3]},
                         {v[8 * k + 4], v[8 * k + 5], v[8 * k + 6]}, v[8 * k + 7]};
    printf("%d\n", tlpg::rows_overlap(t[0], t[1]) ? 1 : 0);
  }
}
"""


@pytest.fixture(scope="module")
def overlaps(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    d = tmp_path_factory.mktemp("overlap")
    (d / "main.hip").write_text(MAIN)
    res = subprocess.run([hipcc, "--offload-host-only", "-std=c++17", "-I", os.path.join(ROOT, "triton-llm_amd", "csrc"),
                          "-I", os.path.join(ROOT, "include"), str(d / "main.hip"), "-o", str(d / "main")],
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr

    def run(cases):
        text = "".join(" ".join(map(str, a + b)) + "\n" for a, b in cases)
        out = subprocess.run([str(d / "main")], input=text, capture_output=True, text=True, check=True).stdout
        return [int(x) for x in out.split()]

    return run


def tensor(base, n, s, row):
    return (base, *n, *s, row)


def bytes_of(t):
    base, n0, n1, n2, s0, s1, s2, row = t
    at = base + np.add.outer(np.add.outer(np.arange(n0) * s0, np.arange(n1) * s1), np.arange(n2) * s2).ravel()
    return set((at[:, None] + np.arange(row)).ravel().tolist())


def test_no_shared_byte_is_missed(overlaps):
    rng = np.random.default_rng(0)
    cases = []
    for _ in range(6000):
        unit = int(rng.choice([1, 4, 12]))
        cases.append(tuple(tensor(4000 + int(rng.integers(0, 60)), rng.integers(1, 4, 3).tolist(),
                                  (unit * rng.integers(0 if unit > 1 else -9, 14, 3)).tolist(), int(rng.integers(1, 9)))
                           for _ in range(2)))
    got = overlaps(cases)
    share = [bool(bytes_of(a) & bytes_of(b)) for a, b in cases]
    assert all(g for g, s in zip(got, share) if s)
    assert sum(not g for g, s in zip(got, share) if not s) > 500  # and many that share none are seen as such


def test_rows_side_by_side(overlaps):
    row, D = 4 * 96, 32  # a token's row of a buffer: q 4 heads, k 2, v 2, o 4 of 32 bytes
    at = lambda first, heads, B=2, S=5: tensor(1 << 20 | first * D, (B, heads, S), (S * row, D, row), D)  # noqa: E731
    q, k, o = at(0, 4), at(4, 2), at(8, 4)
    assert overlaps([(o, q), (o, k), (q, o), (at(3, 4), q), (q, q), (at(3, 1), at(4, 1))]) == [0, 0, 0, 1, 1, 0]
    one = lambda base, heads, S: tensor(base, (1, heads, S), (heads * S * D, S * D, D), D)  # noqa: E731
    assert overlaps([(one(0, 4, 5), one(4 * 5 * D, 4, 5)), (one(0, 4, 5), one(4 * 5 * D - 1, 4, 5))]) == [0, 1]


# ---- the C entries: PTR and its like are never followed, the calls are refused -----------

S3 = _lib.strides(1024, 64, 256)


def c_window(q, k, v, o, os_=S3):
    return _lib.load().tl_window_attention(*(ctypes.c_void_p(x) for x in (q, k, v, o)), None, 0, 1, 4, 4, 8, 8, 64, S3, S3, S3, os_,
                                           0.1, 0, 0, _lib.DTYPE_BF16, None)


def test_c_window_refuses_overlap():
    a, far = 0x100000, 0x200000
    for args in ((a, far, far, a), (far, a, far, a), (far, far, a, a), (a, far, far, a + 2 * 64), (a + 1024, far, far, a)):
        assert c_window(*args) == 1, args


def test_c_paged_refuse_overlap():
    lib = _lib.load()
    a, far, page = 0x100000, 0x4000000, _lib.strides(2 * 16 * 64, 16 * 64, 64)

    def decode(q, k, v, o, os_=S3):
        p = [ctypes.c_void_p(x) for x in (q, k, v)]
        return lib.tl_paged_attention_decode(*p, ctypes.c_void_p(far), 4, 9, 16, ctypes.c_void_p(far), 0, 0, 0, ctypes.c_void_p(o),
                                             ctypes.c_void_p(far), 1 << 30, 2, 4, 2, 64, S3, page, page, os_, 0.1,
                                             _lib.DTYPE_BF16, None)

    def prefill(q, k, v, o):
        p = [ctypes.c_void_p(x) for x in (q, k, v)]
        return lib.tl_paged_attention_prefill(*p, ctypes.c_void_p(far), 4, 9, 16, ctypes.c_void_p(far), None, ctypes.c_void_p(o), None,
                                              0, 2, 3, 4, 2, 64, S3, page, page, S3, 0.1, 0, 0, _lib.DTYPE_BF16, None)

    for args in ((far, a, far, a), (far, far, a, a + 9 * 2 * 16 * 64 * 2 - 1024), (a + 128, far, far, a)):
        assert decode(*args) == 1 and prefill(*args) == 1, args
    assert decode(a, far, far, a, _lib.strides(1024, 128, 256)) == 1  # the same address, another layout
    assert prefill(a, far, far, a) == 1


# ---- on the GPU ----------------------------------------------------------------------

@pytest.mark.gpu
def test_output_beside_the_inputs():
    """q, k, v and o as columns of one buffer's rows."""
    rng = np.random.default_rng(0)
    S, Hq, Hkv, D, dtype = 300, 4, 2, 64, "bfloat16"
    row = (2 * Hq + 2 * Hkv) * D
    x = P.values(rng, (S, row), dtype)
    buf = P.dev(x, dtype)

    def part(first):
        return gpu.DeviceTensor(ctypes.c_void_p(buf.data_ptr() + first * D * 2), (1,), buf.dtype, 2, defer_free=False)

    s = (0, D, row)
    window_attention_strided(part(0), part(Hq), part(Hq + Hkv), part(Hq + 2 * Hkv), batch=1, n_head=Hq, n_kv_head=Hkv, seq_q=S,
                             seq_k=S, d_k=D, q_strides=s, k_strides=s, v_strides=s, o_strides=s, window=40, sinks=2)
    f = on.from_storage(x, dtype).reshape(S, -1, D).transpose(1, 0, 2)
    q = np.ascontiguousarray(x.reshape(S, -1, D).transpose(1, 0, 2)[:Hq])
    want, tol = P.rows_want(q, f[Hq:Hq + Hkv], f[Hq + Hkv:Hq + 2 * Hkv], np.arange(S), True, 40, 2, D ** -0.5, dtype)
    got = P.back(buf, dtype).reshape(S, -1, D).transpose(1, 0, 2)
    np.testing.assert_array_equal(got[:Hq + 2 * Hkv], f[:Hq + 2 * Hkv])
    P.check("beside", got[Hq + 2 * Hkv:], want, tol)


@pytest.mark.gpu
def test_python_calls():
    x = gpu.zeros((1, 4, 64, 64))
    with pytest.raises(RuntimeError, match="window_attention"):
        window_attention(x, gpu.zeros((1, 2, 64, 64)), gpu.zeros((1, 2, 64, 64)), 8, out=x)
    # one token's attention in place of its queries
    rng = np.random.default_rng(1)
    for batch, n in ((2, 40), (64, 300), (1, 3000)):
        q = P.dev(P.values(rng, (batch, 4, 64), "float32"), "float32")
        pages = -(-n // 16)
        pool = [P.dev(P.values(rng, (batch * pages, 2, 16, 64), "float32"), "float32") for _ in "kv"]
        table, lens = P.int32(np.arange(batch * pages).reshape(batch, pages)), P.int32(np.full(batch, n))
        want = gpu.to_host(paged_attention_decode(q, *pool, table, lens, 4, 2))
        paged_attention_decode(q, *pool, table, lens, 4, 2, out=q)
        np.testing.assert_array_equal(gpu.to_host(q), want)
