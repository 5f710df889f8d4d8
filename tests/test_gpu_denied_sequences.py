"""Steps in which the pool has too few pages: sequences that are not granted theirs leave the others' rows, pages and lengths as they
are, also where their row of the table still names pages that others hold now, and go on once there is room."""

import numpy as np
import pytest

from tests.test_gpu_serving_runs import Server
from triton_llm import gpu

pytestmark = pytest.mark.gpu


def step(s, new, ended, granted, name):
    """A step of which `granted` sequences get their pages; their rows are checked, the others' are no tokens."""
    s.load(new, ended)
    before = gpu.to_host(s.lens)
    s.device_step(s.packed)
    slots, _, starts, ends = (gpu.to_host(t) for t in s.out)
    for b, n in enumerate(new):
        at = slice(starts[b], starts[b] + n)
        assert (slots[at] >= 0).all() if granted[b] else (slots[at] == -1).all()
        assert ends[b] == (0 if ended[b] else before[b]) + (n if granted[b] else 0)
    assert gpu.to_host(s.counts)[1] == sum(1 for n, g in zip(new, granted) if n and not g)
    # check() goes through the granted ones' rows alone
    rows, out = s.now, s.o
    keep = np.concatenate([np.arange(starts[b], starts[b] + n) for b, n in enumerate(new) if granted[b]])
    s.now = [x[keep] for x in rows]
    s.expect = [n if g else 0 for n, g in zip(new, granted)]
    data = gpu.to_host(out)
    s.o = gpu.to_device(np.ascontiguousarray(data[keep]), out.dtype)
    s.check(name)
    s.now, s.o = rows, out


@pytest.mark.parametrize("dtype,Hq,Hkv,D", [("float32", 3, 1, 64), ("bfloat16", 6, 2, 128), ("float16", 4, 2, 64)])
def test_a_pool_too_small(dtype, Hq, Hkv, D):
    s = Server(dtype, Hq, Hkv, D, 16, batch=4, max_pages=8, n_pages=6, tokens=160)
    step(s, [40, 20, 50, 0], [0, 0, 0, 0], [1, 1, 0, 1], "third denied")
    step(s, [1, 1, 30, 0], [0, 0, 0, 0], [1, 1, 0, 1], "denied again")
    step(s, [0, 1, 50, 0], [1, 0, 0, 0], [1, 1, 1, 1], "the first's pages go to the third")
    # the first row of the table still names pages that the third sequence holds
    step(s, [33, 1, 1, 7], [0, 0, 0, 0], [0, 1, 1, 0], "first and last denied")
    step(s, [33, 1, 1, 7], [0, 0, 1, 0], [1, 1, 1, 0], "room again")
