"""The paged cache on the GPU against the 64-bit forms.  Positions that a call may not read hold NaN;
tolerances are those derived in tests/_paged.py."""

import numpy as np
import pytest

from oracle import numerics as on
from oracle import paged as op
from tests import _paged as P
from triton_llm import gpu
from triton_llm.kernels import (allocate_kv_pages, copy_kv_pages, paged_attention_decode, paged_attention_prefill,
                                paged_decode_workspace, paged_kv_append, precompute_cos_sin, write_i32)

pytestmark = pytest.mark.gpu
DTYPES = ["float32", "float16", "bfloat16"]


# ---- append -------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,Hq,Hkv,D,page,n_new,rotary,inter,in_place", [
    ("bfloat16", 24, 8, 128, 16, 1, 128, False, True),
    ("float16", 15, 5, 64, 32, 37, 32, True, False),
    ("float32", 9, 3, 64, 16, 19, 64, False, False),
    ("float32", 4, 2, 64, 64, 33, 16, True, True),
    ("bfloat16", 3, 1, 128, 16, 5, 64, False, False),
    ("bfloat16", 4, 4, 64, 16, 3, 0, False, False),
    ("float16", 2, 1, 6, 16, 20, 4, False, False),   # rows of no round size
    ("bfloat16", 2, 1, 10, 16, 20, 6, True, True),
    ("float32", 2, 2, 24, 128, 130, 12, False, True),
    ("float16", 2, 1, 16, 1024, 7, 2, True, False),
])
def test_append(dtype, Hq, Hkv, D, page, n_new, rotary, inter, in_place):
    rng = np.random.default_rng(n_new)
    lens = np.array([0, page - 1, 3 * page - n_new, 7, 2 * page, -2, 1 << 30], np.int32)
    new = np.array([n_new, max(1, n_new // 2), n_new, 0, n_new, n_new, n_new], np.int32)
    B, max_pages = len(lens), 3 + n_new // page
    n_pages = B * max_pages + 2
    table = P.shuffled_table(rng, [max_pages * page] * B, page, max_pages, n_pages)
    table[4, 2] = n_pages      # a page that is not there
    table[1, 1] = -5
    shape = (n_pages, Hkv, page, D)
    kp, vp = P.values(rng, shape, dtype), P.values(rng, shape, dtype)
    q = P.values(rng, (B, n_new, Hq, D), dtype)
    k, v = P.values(rng, (B, n_new, Hkv, D), dtype), P.values(rng, (B, n_new, Hkv, D), dtype)
    rows = max_pages * page - 2  # the table of angles ends before the pages do
    cos, sin = precompute_cos_sin(rows, rotary) if rotary else (None, None)
    before = P.values(rng, q.shape, dtype)
    qo_d = None if in_place else P.dev(before, dtype)
    q_d, kp_d, vp_d = P.dev(q, dtype), P.dev(kp, dtype), P.dev(vp, dtype)
    tab = [gpu.to_device(x) if x is not None else None for x in (cos, sin)]
    out = paged_kv_append(q_d, P.dev(k, dtype), P.dev(v, dtype), kp_d, vp_d, P.int32(table), P.int32(lens), *tab,
                          new_lens=P.int32(new), q_out=qo_d, interleaved=inter)
    want = op.append(q, k, v, kp, vp, table, lens, cos, sin, new, None if in_place else before, inter, dtype)
    if in_place and not rotary:
        want = (q,) + want[1:]
    bits = {2: np.uint16, 4: np.uint32}[kp.dtype.itemsize]
    for name, got, exp in zip(("q", "k", "v"), (out, kp_d, vp_d), want):
        np.testing.assert_array_equal(gpu.to_host(got).view(bits), exp.view(bits), err_msg=name)


def test_append_without_q_or_lens():
    """Three-dimensional tensors, no query, no new_lens, no positions."""
    rng = np.random.default_rng(3)
    kp, vp = P.values(rng, (5, 2, 16, 64), "bfloat16"), P.values(rng, (5, 2, 16, 64), "bfloat16")
    k, v = P.values(rng, (2, 2, 64), "bfloat16"), P.values(rng, (2, 2, 64), "bfloat16")
    table, lens = np.array([[4, 1], [0, 2]], np.int32), np.array([16, 3], np.int32)
    kp_d, vp_d = P.dev(kp, "bfloat16"), P.dev(vp, "bfloat16")
    assert paged_kv_append(None, P.dev(k, "bfloat16"), P.dev(v, "bfloat16"), kp_d, vp_d, P.int32(table), P.int32(lens)) is None
    _, wk, wv = op.append(None, k[:, None], v[:, None], kp, vp, table, lens, dtype="bfloat16")
    np.testing.assert_array_equal(gpu.to_host(kp_d).view(np.uint16), wk)
    np.testing.assert_array_equal(gpu.to_host(vp_d).view(np.uint16), wv)


# ---- one token -----------------------------------------------------------------------

def run_decode(dtype, Hq, Hkv, D, page, lens, window, sinks, len_add=0, scale=None, seed=0, table_edit=None, max_pages=None):
    rng = np.random.default_rng(seed)
    total = np.asarray(lens, np.int64) + len_add
    need = [max(0, int(n)) for n in total]
    max_pages = max_pages or max(1, -(-max(need) // page))
    cap = max_pages * page
    need = [min(n, cap) for n in need]
    n_pages = sum(-(-n // page) for n in need) + 2
    table = P.shuffled_table(rng, need, page, max_pages, n_pages)
    if table_edit:
        table_edit(table, n_pages)
    keep = [op.seen([n - 1], n, window, sinks)[0] for n in need]
    shape = (n_pages, Hkv, page, D)
    kp, vp = P.pool_with(rng, table, keep, shape, dtype), P.pool_with(rng, table, keep, shape, dtype)
    q = P.values(rng, (len(lens), Hq, D), dtype)
    scale = scale if scale is not None else D ** -0.5
    out = gpu.to_device(np.full(q.shape, on.nan_storage(dtype), on.storage_dtype(dtype)), P.H.GPU_DTYPES[dtype])
    paged_attention_decode(P.dev(q, dtype), P.dev(kp, dtype), P.dev(vp, dtype), P.int32(table), P.int32(lens), Hq, Hkv,
                           sm_scale=scale, len_add=len_add, window=window, sinks=sinks, out=out,
                           workspace=paged_decode_workspace(len(lens), Hq, Hkv, cap, D))
    want, tol = P.decode_want(q, np.where(np.isnan(on.from_storage(kp, dtype)), 0, kp).astype(kp.dtype),
                              np.where(np.isnan(on.from_storage(vp, dtype)), 0, vp).astype(vp.dtype), table, total,
                              window, sinks, scale, dtype)
    P.check(f"decode {dtype} {Hq}/{Hkv} d{D} page {page} window {window} sinks {sinks}", P.back(out, dtype), want, tol)


@pytest.fixture(params=["pair", "shares"])
def mode(request, monkeypatch):
    """Short caches take a workgroup a (sequence, KV head), others equal shares of all blocks; the override sends
    every call through the shares."""
    P.H.set_override(monkeypatch, "TRITON_LLM_HIP_DECODE_SHARES", 1 if request.param == "shares" else None)


SHORT = [0, 1, 15, 16, 17, 31, 33, 64, 100, 255, 257]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page,window,sinks", [(16, 0, 0), (32, 20, 3), (256, 1, 0), (16, 64, 16), (64, 50, 40),
                                               (16, 16, 1 << 30), (1024, 1 << 30, 0), (16, 33, 17)])
def test_decode_lengths(mode, dtype, D, page, window, sinks):
    run_decode(dtype, 6, 2, D, page, SHORT, window, sinks)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (4, 2), (4, 1), (5, 1), (6, 1), (14, 2), (8, 1), (12, 1), (17, 1), (9, 9)])
@pytest.mark.parametrize("dtype,D", [("bfloat16", 128), ("float32", 64), ("float16", 64), ("float32", 128)])
def test_decode_groups(mode, Hq, Hkv, dtype, D):
    run_decode(dtype, Hq, Hkv, D, 16, [3, 200, 0, 90], 0, 0)


def test_decode_many_sequences_and_len_add(mode):
    rng = np.random.default_rng(5)
    run_decode("bfloat16", 4, 2, 64, 16, rng.integers(0, 90, 150), 0, 0, len_add=1)
    run_decode("float16", 4, 2, 64, 32, rng.integers(-3, 60, 65), 25, 2, len_add=-2)


def test_decode_long_and_past_the_table():
    run_decode("bfloat16", 3, 1, 128, 64, [9000, 1, 5000], 0, 0)
    run_decode("float32", 3, 1, 64, 16, [9000, 40, 3000], 1500, 4)
    run_decode("float16", 2, 1, 64, 16, [1 << 30, 40, -7], 0, 0, max_pages=5)  # lengths end where the table does


def test_decode_scales(mode):
    for scale in (-0.2, 0.0, 4.0):
        run_decode("float16", 2, 1, 64, 16, [40, 3], 0, 0, scale=scale)


def test_decode_pages_that_are_not_there(mode):
    def edit(table, n_pages):
        table[0, 1], table[0, 4], table[2, :] = -1, n_pages, 2 ** 31 - 1
        table[1, 0] = -2 ** 31
    run_decode("bfloat16", 3, 1, 64, 16, [90, 40, 33], 0, 0, table_edit=edit)
    run_decode("float32", 3, 1, 128, 16, [90, 40, 33], 30, 5, table_edit=edit)


def test_decode_fewer_compute_units(monkeypatch):
    """Shares of many blocks: pairs begin and end inside them, and over several."""
    P.H.set_override(monkeypatch, "TRITON_LLM_HIP_DECODE_SHARES", 1)
    for cus in (1, 3):
        P.H.set_override(monkeypatch, "TRITON_LLM_HIP_MAX_CUS", cus)
        run_decode("bfloat16", 6, 2, 64, 16, [700, 0, 1300, 5, 64], 0, 0)
        run_decode("bfloat16", 6, 2, 64, 16, [700, 0, 1300, 5, 64], 100, 7)


# ---- many tokens ---------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,page,window,sinks", [(64, 16, 0, 0), (128, 32, 0, 0), (64, 16, 40, 3), (128, 128, 100, 0),
                                                 (128, 16, 1, 1), (64, 1024, 130, 70), (64, 32, 1 << 30, 1 << 30)])
def test_prefill(dtype, D, page, window, sinks):
    rng = np.random.default_rng(D + page)
    Hq, Hkv, n_new = 4, 2, 150
    lens = np.array([0, 1, 333, 5, 64, -3], np.int32)
    new = np.array([150, 129, 37, 0, 1, 20], np.int32)
    total = lens + new
    max_pages = -(-int(total.max()) // page)
    n_pages = sum(-(-max(int(t), 0) // page) for t in total) + 2
    table = P.shuffled_table(rng, total, page, max_pages, n_pages)
    keep = [np.arange(max_pages * page) < t for t in total]
    shape = (n_pages, Hkv, page, D)
    kp, vp = P.pool_with(rng, table, keep, shape, dtype), P.pool_with(rng, table, keep, shape, dtype)
    q = P.values(rng, (len(lens), n_new, Hq, D), dtype)
    before = P.values(rng, q.shape, dtype)
    out = P.dev(before, dtype)
    paged_attention_prefill(P.dev(q, dtype), P.dev(kp, dtype), P.dev(vp, dtype), P.int32(table), P.int32(lens), Hq, Hkv,
                            new_lens=P.int32(new), window=window, sinks=sinks, out=out)
    got = P.back(out, dtype)
    for b, (n, m) in enumerate(zip(lens, new)):
        np.testing.assert_array_equal(got[b, m:], on.from_storage(before[b, m:], dtype))  # rows behind the tokens
        if m == 0:
            continue
        k, there = op.gather(on.from_storage(kp, dtype), table[b], max(int(n + m), 1))
        v, _ = op.gather(on.from_storage(vp, dtype), table[b], max(int(n + m), 1))
        want, tol = P.rows_want(q[b, :m].transpose(1, 0, 2), k, v, n + np.arange(m), there, window, sinks, D ** -0.5, dtype)
        P.check(f"prefill {dtype} d{D} page {page} window {window} sequence {b}", got[b, :m].transpose(1, 0, 2), want, tol)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prefill_pages_that_are_not_there(dtype):
    rng = np.random.default_rng(8)
    Hq, Hkv, D, page, n_new = 2, 1, 64, 16, 70
    lens = np.array([60, 10, 0], np.int32)
    total = lens + n_new
    table = P.shuffled_table(rng, total, page, 7, 30)  # sequence 0 goes on behind its last page
    table[0, 2], table[0, 5], table[1, :2], table[2, :] = -1, 30, 2 ** 31 - 1, -1
    keep = [np.arange(7 * page) < t for t in total]
    kp, vp = (P.pool_with(rng, table, keep, (30, Hkv, page, D), dtype) for _ in range(2))
    q = P.values(rng, (3, n_new, Hq, D), dtype)
    out = paged_attention_prefill(P.dev(q, dtype), P.dev(kp, dtype), P.dev(vp, dtype), P.int32(table), P.int32(lens), Hq, Hkv)
    got = P.back(out, dtype)
    for b in range(3):
        n = min(int(total[b]), 7 * page)
        k, there = op.gather(on.from_storage(kp, dtype), table[b], n)
        v, _ = op.gather(on.from_storage(vp, dtype), table[b], n)
        want, tol = P.rows_want(q[b].transpose(1, 0, 2), k, v, lens[b] + np.arange(n_new), there, 0, 0, D ** -0.5, dtype)
        P.check(f"prefill without pages {dtype} sequence {b}", got[b].transpose(1, 0, 2), want, tol)


@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 0), (30, 5), (1000, 2), ((1 << 31) - 1, 0)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_prefill_past_the_table(dtype, window, sinks):
    """Queries behind the last page, some by more than the window: they see what there is."""
    rng = np.random.default_rng(12)
    Hq, Hkv, D, page, n_new, cap = 2, 1, 64, 16, 140, 112
    lens = np.array([100, 200, 2 ** 31 - 1, 0, -2 ** 31], np.int32)
    table = rng.permutation(30)[:7][None].repeat(5, 0).astype(np.int32)
    kp, vp = P.values(rng, (30, Hkv, page, D), dtype), P.values(rng, (30, Hkv, page, D), dtype)
    q = P.values(rng, (5, n_new, Hq, D), dtype)
    out = paged_attention_prefill(P.dev(q, dtype), P.dev(kp, dtype), P.dev(vp, dtype), P.int32(table), P.int32(lens), Hq, Hkv,
                                  window=window, sinks=sinks)
    got = P.back(out, dtype)
    k, there = op.gather(on.from_storage(kp, dtype), table[0], cap)
    v, _ = op.gather(on.from_storage(vp, dtype), table[0], cap)
    for b in (0, 1, 3):
        want, tol = P.rows_want(q[b].transpose(1, 0, 2), k, v, lens[b] + np.arange(n_new), there, window, sinks, D ** -0.5, dtype)
        P.check(f"prefill past the table {dtype} window {window} sequence {b}", got[b].transpose(1, 0, 2), want, tol)
    assert (got[4] == 0).all()
    if window == 30 and sinks == 0:
        assert (got[2] == 0).all()
    else:  # the window hides nothing or all but the sinks
        far = np.full(n_new, cap if window in (0, (1 << 31) - 1) else cap + window)
        want, tol = P.rows_want(q[2].transpose(1, 0, 2), k, v, far, there, window, sinks, D ** -0.5, dtype)
        P.check(f"prefill far past the table {dtype} window {window}", got[2].transpose(1, 0, 2), want, tol)


# ---- pools of more than 4 GiB ------------------------------------------------------------

def test_pages_beyond_32_bit_offsets():
    """A 5 GiB pool: the last pages are written, read by one token and by many, and copied."""
    rng = np.random.default_rng(9)
    dtype, Hq, Hkv, D, page, n = "bfloat16", 2, 1, 128, 1024, 70
    n_pages = 5 * (1 << 30) // (page * D * 2)
    kp, vp = allocate_kv_pages(n_pages, Hkv, page, D, P.H.GPU_DTYPES[dtype], zero=False)
    q, k, v = P.values(rng, (1, n, Hq, D), dtype), P.values(rng, (1, n, Hkv, D), dtype), P.values(rng, (1, n, Hkv, D), dtype)
    kf, vf = (on.from_storage(x, dtype)[0].transpose(1, 0, 2) for x in (k, v))
    want, tol = P.rows_want(q[0].transpose(1, 0, 2), kf, vf, np.arange(n), np.ones(n, bool), 0, 0, D ** -0.5, dtype)
    q_d = P.dev(q, dtype)
    paged_kv_append(q_d, P.dev(k, dtype), P.dev(v, dtype), kp, vp, P.int32([[n_pages - 1]]), P.int32([0]))
    copy_kv_pages([kp, vp], [n_pages - 1], [n_pages - 3])
    for at in (n_pages - 1, n_pages - 3):
        table = P.int32([[at]])
        out = paged_attention_prefill(q_d, kp, vp, table, P.int32([0]), Hq, Hkv)
        P.check(f"prefill page {at}", P.back(out, dtype)[0].transpose(1, 0, 2), want, tol)
        one = paged_attention_decode(P.dev(q[:, -1], dtype), kp, vp, table, P.int32([n]), Hq, Hkv)
        P.check(f"decode page {at}", P.back(one, dtype)[0], want[:, -1], tol[:, -1])


# ---- copies and writes ---------------------------------------------------------------------

@pytest.mark.parametrize("dtype,layers,shape,moved", [("float32", 2, (9, 3, 16, 64), 3), ("bfloat16", 66, (700, 1, 16, 2), 300),
                                                      ("float16", 1, (6, 8, 64, 128), 3), ("bfloat16", 3, (5, 5, 32, 6), 1)])
def test_copy_pages(dtype, layers, shape, moved):
    rng = np.random.default_rng(moved)
    host = [P.values(rng, shape, dtype) for _ in range(layers)]
    pools = [P.dev(x, dtype) for x in host]
    order = rng.permutation(shape[0])
    src, dst = order[:moved], order[-moved:]
    copy_kv_pages(pools, src, dst)
    for x, t in zip(host, pools):
        x[dst] = x[src]
        np.testing.assert_array_equal(gpu.to_host(t).view(np.uint8), x.view(np.uint8))
    if moved > 1:  # one page to many
        copy_kv_pages(pools[:1], [int(dst[0])] * (moved - 1), src[:moved - 1])
        host[0][src[:moved - 1]] = host[0][dst[0]]
        np.testing.assert_array_equal(gpu.to_host(pools[0]).view(np.uint8), host[0].view(np.uint8))


def test_write_i32():
    rng = np.random.default_rng(1)
    x = rng.integers(-9, 9, (40, 20)).astype(np.int32)
    t = gpu.to_device(x)
    at = rng.permutation(800)[:600]
    val = rng.integers(-2 ** 31, 2 ** 31, 600)
    write_i32(t, at, val)
    x.ravel()[at] = val
    np.testing.assert_array_equal(gpu.to_host(t), x)


# ---- graphs ---------------------------------------------------------------------------------

def test_captured_step_replays():
    """Append, attention, a page copy and a table write in one graph; every replay equals the eager
    calls, with eager work between, and a second graph shares the workspace."""
    rng = np.random.default_rng(11)
    dtype, Hq, Hkv, D, page, B = "bfloat16", 6, 2, 64, 16, 5
    lens = np.array([3, 40, 0, 100, 15], np.int32)
    table = P.shuffled_table(rng, lens + 1, page, 8, 30)
    kp, vp = P.values(rng, (30, Hkv, page, D), dtype), P.values(rng, (30, Hkv, page, D), dtype)
    q, k, v = P.values(rng, (B, Hq, D), dtype), P.values(rng, (B, Hkv, D), dtype), P.values(rng, (B, Hkv, D), dtype)
    cos, sin = (gpu.to_device(x) for x in precompute_cos_sin(128, D))
    free = np.setdiff1d(np.arange(30), table)[:1]
    src = int(table[1, 0])

    def state():
        return dict(kp=P.dev(kp, dtype), vp=P.dev(vp, dtype), q=P.dev(q, dtype), k=P.dev(k, dtype), v=P.dev(v, dtype),
                    qo=P.dev(q, dtype), out=P.dev(q, dtype), table=P.int32(table), lens=P.int32(lens), count=P.int32([0, 0]))

    ws = paged_decode_workspace(B, Hq, Hkv, 128, D)

    def step(s):
        paged_kv_append(s["q"], s["k"], s["v"], s["kp"], s["vp"], s["table"], s["lens"], cos, sin, q_out=s["qo"])
        paged_attention_decode(s["qo"], s["kp"], s["vp"], s["table"], s["lens"], Hq, Hkv, len_add=1, out=s["out"], workspace=ws)
        copy_kv_pages([s["kp"], s["vp"]], [src], free)
        write_i32(s["count"], [1], [7])

    eager = state()
    step(eager)
    want = {n: gpu.to_host(eager[n]) for n in ("out", "kp", "vp", "qo", "count")}
    graphs = []
    for _ in range(2):
        s = state()
        gpu.synchronize()
        with gpu.capture() as g:
            step(s)
        graphs.append((g, s))
    for i in range(3):
        for g, s in graphs:
            s["kp"].from_numpy(kp)
            s["out"].from_numpy(np.zeros_like(q))
            g.replay()
            step(eager)  # eager work on the same workspace
            for n, x in want.items():
                np.testing.assert_array_equal(gpu.to_host(s[n]).view(np.uint8), x.view(np.uint8), err_msg=f"{n} replay {i}")


@pytest.mark.parametrize("dtype,D,batch,cus", [("bfloat16", 64, 70, None), ("float32", 64, 70, 200), ("float16", 128, 3, 2), ("bfloat16", 64, 5, 7)])
def test_prefill_divided_keys(monkeypatch, dtype, D, batch, cus):
    """Few rows on long and short prefixes: the keys are shared by workgroups, sequences without tokens among them."""
    P.H.set_override(monkeypatch, "TRITON_LLM_HIP_MAX_CUS", cus)
    rng = np.random.default_rng(batch)
    Hq, Hkv, page, n_new = 2, 1, 32, 5
    lens = rng.integers(0, 1500, batch).astype(np.int32)
    lens[::7] = 0
    new = rng.integers(0, n_new + 1, batch).astype(np.int32)
    new[0] = n_new
    total = lens + new
    max_pages = 50
    n_pages = sum(-(-int(t) // page) for t in total) + 2
    table = P.shuffled_table(rng, total, page, max_pages, n_pages)
    keep = [np.arange(max_pages * page) < t for t in total]
    kp, vp = (P.pool_with(rng, table, keep, (n_pages, Hkv, page, D), dtype) for _ in range(2))
    q = P.values(rng, (batch, n_new, Hq, D), dtype)
    before = P.values(rng, q.shape, dtype)
    kp_d, vp_d = P.dev(kp, dtype), P.dev(vp, dtype)
    for window, sinks in ((0, 0), (700, 5)):
        out = P.dev(before, dtype)
        paged_attention_prefill(P.dev(q, dtype), kp_d, vp_d, P.int32(table), P.int32(lens), Hq, Hkv, new_lens=P.int32(new),
                                window=window, sinks=sinks, out=out)
        got = P.back(out, dtype)
        for b in range(batch):
            n, m = int(lens[b]), int(new[b])
            np.testing.assert_array_equal(got[b, m:], on.from_storage(before[b, m:], dtype))
            if m == 0:
                continue
            k, there = op.gather(on.from_storage(kp, dtype), table[b], n + m)
            v, _ = op.gather(on.from_storage(vp, dtype), table[b], n + m)
            want, tol = P.rows_want(q[b, :m].transpose(1, 0, 2), k, v, n + np.arange(m), there, window, sinks, D ** -0.5, dtype)
            P.check(f"divided {dtype} sequence {b} {n}+{m} window {window}", got[b, :m].transpose(1, 0, 2), want, tol)


@pytest.mark.parametrize("dtype,D,lens", [("float32", 64, [700]), ("bfloat16", 128, [1500, 3, 900, 0]),
                                          ("float16", 64, [40] * 70 + [2000])])
def test_shared_positions_replay(monkeypatch, dtype, D, lens):
    """Sequences shared by workgroups: from a workspace that holds anything, eager and replayed with other calls on the same
    workspace between, always the same bits."""
    P.H.set_override(monkeypatch, "TRITON_LLM_HIP_DECODE_SHARES", 1)
    rng = np.random.default_rng(21)
    Hq, Hkv, page = 6, 2, 16
    lens = np.array(lens, np.int32)
    max_pages = 2048 // page
    n_pages = int(sum(-(-int(n) // page) for n in lens)) + 1
    table = P.shuffled_table(rng, lens, page, max_pages, n_pages)
    kp, vp = (P.dev(P.values(rng, (n_pages, Hkv, page, D), dtype), dtype) for _ in range(2))
    q = P.dev(P.values(rng, (len(lens), Hq, D), dtype), dtype)
    t_d, l_d, short = P.int32(table), P.int32(lens), P.int32(np.minimum(lens, 333))
    ws = gpu.to_device(np.full(1 << 26, 0xFF, np.uint8))

    def call(n, **kw):
        return paged_attention_decode(q, kp, vp, t_d, n, Hq, Hkv, workspace=ws, **kw)

    first = P.back(call(l_d), dtype)
    plain = P.back(paged_attention_decode(q, kp, vp, t_d, l_d, Hq, Hkv), dtype)
    np.testing.assert_array_equal(plain, first)
    assert np.isfinite(first).all()
    out = P.dev(np.zeros(q.shape, on.storage_dtype(dtype)), dtype)
    gpu.synchronize()
    with gpu.capture() as g:
        call(l_d, out=out)
    for i in range(4):
        out.from_numpy(np.full(q.shape, on.nan_storage(dtype), on.storage_dtype(dtype)))
        if i % 2:
            call(short)
        g.replay()
        np.testing.assert_array_equal(P.back(out, dtype), first)
        np.testing.assert_array_equal(P.back(call(l_d), dtype), first)
