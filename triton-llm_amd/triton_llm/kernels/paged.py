"""A KV cache in pages: append, attention and page copies (additive API).

The reference keeps one contiguous cache per sequence (smollm2_triton/model.py:190-225);
:mod:`~triton_llm.kernels.decode` keeps such caches on the GPU.  Here a layer's K and V are
pools of pages ``(n_pages, n_kv_head, page_size, d_k)`` and a table
``page_table`` ``(batch, max_pages)`` int32 names each sequence's pages in order, so that
sequences of any length share one pool, and a common prefix is held once:

* :func:`allocate_kv_pages` -- the two pools of a layer;
* :func:`paged_kv_append` -- rotary positions on q and k, k and v written at
  ``cache_lens[b] + s``;
* :func:`paged_attention_decode` -- one new token per sequence over its pages;
* :func:`paged_attention_prefill` -- many new tokens per sequence over their
  pages, a prefix that is there already among them;
* :func:`copy_kv_pages` -- pages copied in every layer at once, for forks and
  compaction.

``page_size`` is a power of two from 16 to 1024.  A table entry outside
``[0, n_pages)`` (-1, by convention) names no page: its positions are not written,
and no query sees them.  ``cache_lens`` is an int32 device array of the tokens
cached before the call; nothing here changes it, and nothing synchronises.
With ``window`` > 0 a query sees the last ``window`` positions up to its own
and the first ``sinks`` of the sequence; 0 means all up to its own.
"""

from __future__ import annotations

import ctypes
import functools
import math
import operator

import numpy as np

from triton_llm import _lib, gpu
from ._common import default_scale, launch, same_dtype, scratch

MIN_PAGE, MAX_PAGE = 16, 1024


def check_page_size(page_size: int) -> None:
    if not (MIN_PAGE <= page_size <= MAX_PAGE and page_size & (page_size - 1) == 0):
        raise ValueError(f"page_size must be a power of 2 in [{MIN_PAGE}, {MAX_PAGE}], got {page_size}")


def allocate_kv_pages(n_pages: int, n_kv_head: int, page_size: int, d_k: int, dtype=np.float32, zero: bool = True):
    """(k_pages, v_pages), each ``(n_pages, n_kv_head, page_size, d_k)`` on the GPU."""
    if n_pages <= 0 or n_kv_head <= 0 or d_k <= 0:
        raise ValueError(f"pool dims must be positive, got n_pages={n_pages} n_kv_head={n_kv_head} d_k={d_k}")
    check_page_size(page_size)
    gpu.dtype_code(dtype)
    alloc = gpu.zeros if zero else gpu.allocate
    shape = (n_pages, n_kv_head, page_size, d_k)
    return alloc(shape, dtype), alloc(shape, dtype)


# The checks of shapes and what follows from them (strides as the C entries take them) are kept
# per combination of shapes: a decode step of a serving loop comes with the same ones every time, and
# putting them together costs more than the launch.  Types are checked in every call.

def _is_int32(t) -> bool:
    return t.dtype.char == "i"


def dtype_code_of(*tensors) -> int:
    """Dtype code shared by all tensors; ValueError if they differ (same_dtype, without its pass over the
    names where every tensor has the very same dtype object)."""
    dt = tensors[0].dtype
    for t in tensors:
        if t.dtype is not dt:
            return same_dtype(*tensors)
    return _BF16 if dt is gpu.bfloat16 else gpu.dtype_code(dt)


_BF16 = _lib.DTYPE_BF16


def _ptr(t):
    return None if t is None else t.ptr


def _check_pool(k_shape, v_shape):
    if len(k_shape) != 4 or k_shape != v_shape:
        raise ValueError(f"k_pages/v_pages must be matching 4-D (n_pages, n_kv_head, page_size, d_k), "
                         f"got {k_shape} and {v_shape}")
    if min(k_shape) <= 0:
        raise ValueError(f"pool dims must be positive, got {k_shape}")
    check_page_size(k_shape[2])
    return k_shape


def _check_table(table_shape, lens_shape, new_lens_shape, page_size, most):
    if len(table_shape) != 2 or table_shape[1] < 1:
        raise ValueError(f"page_table must be int32 (batch, max_pages), got {table_shape}")
    batch, max_pages = table_shape
    if max_pages * page_size > most:
        raise ValueError(f"{max_pages} pages of {page_size} exceed {most} positions")
    for name, shape in (("cache_lens", lens_shape), ("new_lens", new_lens_shape)):
        if shape is not None and shape != (batch,):
            raise ValueError(f"{name} must be int32 of shape ({batch},), got {shape}")
    return batch, max_pages


def _check_int32(page_table, cache_lens, new_lens=None):
    if page_table.dtype.char == cache_lens.dtype.char == "i" and (new_lens is None or new_lens.dtype.char == "i"):
        return
    for name, t in (("page_table", page_table), ("cache_lens", cache_lens), ("new_lens", new_lens)):
        if t is not None and not _is_int32(t):
            raise ValueError(f"{name} must be int32, got {gpu.dtype_name(t.dtype)} {t.shape}")


def _check_heads(n_head, n_kv_head, n_kv, d_k):
    if n_kv != n_kv_head:
        raise ValueError(f"pool has {n_kv} KV heads, n_kv_head={n_kv_head}")
    if n_head <= 0 or n_kv_head <= 0 or n_head % n_kv_head:
        raise ValueError(f"n_head ({n_head}) must be a positive multiple of n_kv_head ({n_kv_head})")
    if d_k not in (64, 128):
        raise ValueError(f"paged attention supports d_k in (64, 128), got {d_k}")


def check_window(window: int, sinks: int) -> None:
    if not (0 <= window < 1 << 31 and 0 <= sinks < 1 << 31):
        raise ValueError(f"window and sinks must be >= 0 and fit in int32, got {window} and {sinks}")


def _same_output(out, q):
    if out is None:
        return gpu.allocate(q.shape, q.dtype)
    if out.shape != q.shape or (out.dtype is not q.dtype and gpu.dtype_name(out.dtype) != gpu.dtype_name(q.dtype)):
        raise ValueError(f"out must be like q, {q.shape} {gpu.dtype_name(q.dtype)}, got {out.shape} "
                         f"{gpu.dtype_name(out.dtype)}")
    return out


def _shape(t):
    return None if t is None else t.shape


@functools.lru_cache(maxsize=1024)
def _append_plan(pool, v_pool, table, lens, new_lens, k, v, q, cos, sin):
    """Strides and sizes of an append by its shapes: the C entry's arguments in their order."""
    n_pages, n_kv, page_size, d_k = _check_pool(pool, v_pool)
    batch, max_pages = _check_table(table, lens, new_lens, page_size, (1 << 31) - 1)
    if len(k) not in (3, 4):
        raise ValueError(f"k_new must be 3-D or 4-D, got {k}")
    n_new = 1 if len(k) == 3 else k[1]
    want = (batch, n_kv, d_k) if len(k) == 3 else (batch, n_new, n_kv, d_k)
    if k != want:
        raise ValueError(f"k_new shape {k} is not {want} (table {table}, pool {pool})")
    if v != want:
        raise ValueError(f"v_new shape {v} != k_new shape {k}")
    if d_k % 2:
        raise ValueError(f"d_k must be even, got {d_k}")
    n_head = 0
    if q is not None:
        if len(q) != len(want) or q[:-2] != want[:-2] or q[-1] != d_k:
            raise ValueError(f"q shape {q} does not match k_new {k}")
        n_head = q[-2]
        if n_head <= 0 or n_head % n_kv:
            raise ValueError(f"n_head ({n_head}) must be a positive multiple of n_kv_head ({n_kv})")
    if (cos is None) != (sin is None):
        raise ValueError("cos_dev and sin_dev must both be given or both be None")
    if cos is not None and (cos != sin or len(cos) != 2 or not 1 <= cos[1] <= d_k // 2):
        raise ValueError(f"cos/sin tables must be float32 (rows, r // 2) with r <= {d_k}, got {cos} and {sin}")
    rows, rotary = (0, 0) if cos is None else (cos[0], 2 * cos[1])
    q_str = _lib.strides(n_new * n_head * d_k, n_head * d_k, d_k)
    kv_str = _lib.strides(n_new * n_kv * d_k, n_kv * d_k, d_k)
    p_str = _lib.strides(n_kv * page_size * d_k, page_size * d_k, d_k)
    return ((max_pages, n_pages, page_size), (rows, rotary),
            (batch, n_new, n_head, n_kv, d_k, q_str, q_str, kv_str, kv_str, p_str, p_str))


def paged_kv_append(q_dev, k_new, v_new, k_pages, v_pages, page_table, cache_lens, cos_dev=None, sin_dev=None,
                    new_lens=None, q_out=None, interleaved: bool = False):
    """Rotate q and k_new, write k and v into the pages at positions ``cache_lens[b] + s``.

    q_dev: ``(batch, n_new, n_head, d_k)`` or ``(batch, n_head, d_k)`` (n_new = 1), or
    None; k_new / v_new: ``(batch, n_new, n_kv_head, d_k)`` or ``(batch, n_kv_head, d_k)``.
    cos/sin: float32 ``(rows, r // 2)`` tables for the first r <= d_k features of a
    head, in pairs (i, i + r/2), or (2i, 2i + 1) with ``interleaved``; None: no
    positions.  ``new_lens`` (int32, ``(batch,)``): how many of a padded batch's n_new rows are
    tokens; the rows behind them are not written.  q goes to ``q_out`` (default: in
    place), which is returned.  Tokens past the table, past cos/sin or without a page
    are skipped, q row and all.  Sequences that share a page may not append to it in
    one call.
    """
    _check_int32(page_table, cache_lens, new_lens)
    pages, tables, sizes = _append_plan(k_pages.shape, v_pages.shape, page_table.shape, cache_lens.shape,
                                        _shape(new_lens), k_new.shape, v_new.shape, _shape(q_dev), _shape(cos_dev),
                                        _shape(sin_dev))
    if q_dev is None:
        if q_out is not None:
            raise ValueError("q_out is given without q_dev")
        code = dtype_code_of(k_new, v_new, k_pages, v_pages)
    else:
        q_out = q_dev if q_out is None else _same_output(q_out, q_dev)
        code = dtype_code_of(k_new, v_new, k_pages, v_pages, q_dev)
    if cos_dev is not None and not cos_dev.dtype.char == sin_dev.dtype.char == "f":
        raise ValueError(f"cos/sin tables must be float32, got {cos_dev.dtype} and {sin_dev.dtype}")
    launch(gpu.runtime().tl_paged_kv_append, _ptr(q_dev), _ptr(q_out), k_new.ptr, v_new.ptr, k_pages.ptr,
           v_pages.ptr, page_table.ptr, *pages, cache_lens.ptr, _ptr(new_lens), _ptr(cos_dev), _ptr(sin_dev), *tables,
           1 if interleaved else 0, *sizes, code, None, what="paged_kv_append")
    return q_out


def paged_decode_workspace(batch: int, n_head: int, n_kv_head: int, max_ctx: int, d_k: int):
    """A workspace of :func:`paged_attention_decode`, reusable by consecutive calls on the
    library stream (calls that overlap in time need one each).  Its size goes by the heads alone."""
    if n_head <= 0 or n_kv_head <= 0 or n_head % n_kv_head:
        raise ValueError(f"n_head ({n_head}) must be a positive multiple of n_kv_head ({n_kv_head})")
    return gpu.allocate((gpu.runtime().tl_paged_decode_workspace_bytes(n_head, n_kv_head, d_k),), np.uint8)


@gpu.plan_cache(1024)
def _attention_plan(pool, v_pool, table, lens, new_lens, q, n_head, n_kv_head, window, sinks, prefill):
    """Strides and sizes of an attention call by its shapes."""
    n_pages, n_kv, page_size, d_k = _check_pool(pool, v_pool)
    batch, max_pages = _check_table(table, lens, new_lens, page_size, 1 << 30 if prefill else (1 << 31) - 1)
    _check_heads(n_head, n_kv_head, n_kv, d_k)
    check_window(window, sinks)
    p_str = _lib.strides(n_kv * page_size * d_k, page_size * d_k, d_k)
    pages = (max_pages, n_pages, page_size)
    if prefill:
        if len(q) != 4 or q[0] != batch or q[2:] != (n_head, d_k):
            raise ValueError(f"q shape {q} is not (batch={batch}, n_new, n_head={n_head}, d_k={d_k})")
        q_str = _lib.strides(q[1] * n_head * d_k, d_k, n_head * d_k)  # {batch, head, seq}
        ws = [_lib.load().tl_window_workspace_bytes(batch, n_head, n_kv_head, q[1], max_pages * page_size, d_k, window,
                                                    sinks, code) for code in range(3)]  # by dtype code
        return pages, (batch, q[1], n_head, n_kv_head, d_k, q_str, p_str, p_str, q_str), ws
    if math.prod(q) != batch * n_head * d_k:
        raise ValueError(f"q shape {q} is not (batch={batch}, n_head={n_head}, d_k={d_k})")
    q_str = _lib.strides(n_head * d_k, d_k)
    return pages, (batch, n_head, n_kv_head, d_k, q_str, p_str, p_str, q_str)


@functools.lru_cache(maxsize=64)
def _decode_workspace_bytes(n_head: int, n_kv_head: int, d_k: int) -> int:
    return _lib.load().tl_paged_decode_workspace_bytes(n_head, n_kv_head, d_k)


def paged_attention_decode(q_dev, k_pages, v_pages, page_table, cache_lens, n_head: int, n_kv_head: int,
                           sm_scale: float | None = None, len_add: int = 0, window: int = 0, sinks: int = 0,
                           out=None, workspace=None):
    """One query per sequence, ``(batch, n_head, d_k)``, over ``cache_lens[b] + len_add`` positions.

    Query head h reads KV head ``h // (n_head // n_kv_head)``.  A sequence without
    visible positions gives zeros.  Hidden positions are not read.
    """
    _check_int32(page_table, cache_lens)
    pages, sizes = _attention_plan(k_pages.shape, v_pages.shape, page_table.shape, cache_lens.shape, None,
                                   q_dev.shape, n_head, n_kv_head, window, sinks, False)
    code = dtype_code_of(q_dev, k_pages, v_pages)
    out = _same_output(out, q_dev)
    d_k = k_pages.shape[3]
    if sm_scale is None:
        sm_scale = default_scale(d_k)
    ws = scratch(_decode_workspace_bytes(n_head, n_kv_head, d_k), workspace, key="paged_decode")
    launch(gpu.runtime().tl_paged_attention_decode, q_dev.ptr, k_pages.ptr, v_pages.ptr, page_table.ptr, *pages,
           cache_lens.ptr, int(len_add), int(window), int(sinks), out.ptr, ws.ptr, ws.nbytes, *sizes, float(sm_scale),
           code, None, what="paged_attention_decode")
    return out


def paged_prefill_workspace_bytes(batch: int, n_head: int, n_kv_head: int, n_new: int, max_ctx: int, d_k: int, dtype,
                                  window: int = 0, sinks: int = 0, host_new_lens=None) -> int:
    """Bytes of a ``workspace`` for :func:`paged_attention_prefill` (0: none is used), max_ctx the positions that a table
    holds.  With ``host_new_lens`` for that call with these counts."""
    _check_heads(n_head, n_kv_head, n_kv_head, d_k)
    check_window(window, sinks)
    need = _lib.load().tl_paged_prefill_workspace_bytes
    dims = (batch, n_head, n_kv_head, n_new, max_ctx, d_k, window, sinks, gpu.dtype_code(dtype))
    most = need(None, *dims)
    return most if host_new_lens is None else max(most, need(_host_counts(host_new_lens, batch), *dims))


def paged_attention_prefill(q_dev, k_pages, v_pages, page_table, cache_lens, n_head: int, n_kv_head: int,
                            new_lens=None, sm_scale: float | None = None, window: int = 0, sinks: int = 0, out=None,
                            workspace=None, host_new_lens=None):
    """Queries ``(batch, n_new, n_head, d_k)`` at positions ``cache_lens[b] + i`` over the pages.

    The new tokens' own k and v are appended before.  ``new_lens`` as in :func:`paged_kv_append`: rows
    behind a sequence's tokens are left as they were.  ``host_new_lens``: the same numbers on the host, where the program has
    them (a sequence of int or a ctypes array): how the work is shared goes by them, and by n_new for every sequence
    otherwise, which is slow where few of a batch's sequences have many tokens.  They may not be less than
    ``new_lens``'s (rows would be left as they were); a captured call goes without them.
    """
    _check_int32(page_table, cache_lens, new_lens)
    pages, sizes, ws_bytes = _attention_plan(k_pages.shape, v_pages.shape, page_table.shape, cache_lens.shape,
                                             _shape(new_lens), q_dev.shape, n_head, n_kv_head, window, sinks, True)
    code = dtype_code_of(q_dev, k_pages, v_pages)
    out = _same_output(out, q_dev)
    need = ws_bytes[code]
    if host_new_lens is not None:
        if new_lens is None:
            raise ValueError("host_new_lens is given without new_lens")
        host_new_lens = _host_counts(host_new_lens, sizes[0])
        # the plan without the counts has its room too: a captured call goes by that
        need = max(need, _lib.load().tl_paged_prefill_workspace_bytes(
            host_new_lens, sizes[0], n_head, n_kv_head, sizes[1], pages[0] * pages[2], sizes[4], window, sinks, code))
    ws = scratch(need, workspace, key="window")
    if sm_scale is None:
        sm_scale = default_scale(k_pages.shape[3])
    launch(gpu.runtime().tl_paged_attention_prefill_counted, q_dev.ptr, k_pages.ptr, v_pages.ptr, page_table.ptr, *pages,
           cache_lens.ptr, _ptr(new_lens), host_new_lens, out.ptr, _ptr(ws), ws.nbytes if ws is not None else 0, *sizes,
           float(sm_scale), int(window), int(sinks), code, None, what="paged_attention_prefill")
    return out


def _host_counts(counts, batch: int):
    """An int32 ctypes array of a batch's counts."""
    if not isinstance(counts, ctypes.Array):
        counts = _numbers(counts)
        if counts and not (min(counts) >= -(1 << 31) and max(counts) < 1 << 31):
            raise ValueError("host_new_lens must fit in int32")
        counts = (ctypes.c_int32 * len(counts))(*counts)
    if len(counts) != batch or counts._type_ is not ctypes.c_int32:
        raise ValueError(f"host_new_lens must hold {batch} int32 numbers, got {len(counts)}")
    return counts


def copy_kv_pages(caches, src, dst) -> None:
    """Page ``dst[i]`` = page ``src[i]`` in every pool of ``caches``.

    caches: pools ``(n_pages, n_kv_head, page_size, d_k)`` of one shape and dtype (the K and V
    of every layer).  src / dst: page numbers on the host; no page may be a destination
    twice, or source and destination.  The numbers travel with the launch: nothing
    synchronises, and a captured graph replays the same copies.
    """
    caches = list(caches)
    src, dst = _numbers(src), _numbers(dst)
    n = len(src)
    if n != len(dst):
        raise ValueError(f"{n} source pages, {len(dst)} destinations")
    if not caches or n == 0:
        return
    shape, dtype = caches[0].shape, caches[0].dtype
    if len(shape) != 4 or min(shape) <= 0:
        raise ValueError(f"pools must be 4-D (n_pages, n_kv_head, page_size, d_k), got {shape}")
    check_page_size(shape[2])
    gpu.dtype_code(dtype)
    for c in caches:
        if c.shape != shape or (c.dtype is not dtype and gpu.dtype_name(c.dtype) != gpu.dtype_name(dtype)):
            raise ValueError(f"pools differ: {shape} {gpu.dtype_name(dtype)} and {c.shape} {gpu.dtype_name(c.dtype)}")
    if min(src) < 0 or min(dst) < 0 or max(src) >= shape[0] or max(dst) >= shape[0]:
        raise ValueError(f"page numbers must be in [0, {shape[0]})")
    to = set(dst)
    if len(to) != n:
        raise ValueError("a page is a destination twice")
    if not to.isdisjoint(src):
        raise ValueError("a page is source and destination")
    page_bytes = shape[1] * shape[2] * shape[3] * dtype.itemsize
    bases = (ctypes.c_void_p * len(caches)).from_buffer_copy(b"".join([c.ptr for c in caches]))
    launch(gpu.runtime().tl_copy_pages, bases, len(caches), page_bytes, page_bytes, shape[0], (ctypes.c_int32 * n)(*src),
           (ctypes.c_int32 * n)(*dst), n, None, what="copy_kv_pages")


def _numbers(x) -> list:
    """Whole numbers of a sequence or array, as a list of int."""
    if isinstance(x, np.ndarray):
        if x.dtype.kind not in "iu":
            raise ValueError(f"expected whole numbers, got {x.dtype}")
        return x.ravel().tolist()
    return [operator.index(i) for i in x]


def write_i32(dst, index, value) -> None:
    """``dst.flat[index[i]] = value[i]`` for a device int32 tensor, the values on the host: no
    upload, no synchronisation (page table entries, lengths).  Indices must be distinct."""
    if not _is_int32(dst):
        raise ValueError(f"dst must be int32, got {gpu.dtype_name(dst.dtype)}")
    index, value = _numbers(index), _numbers(value)
    n = len(index)
    if n != len(value):
        raise ValueError(f"{n} indices, {len(value)} values")
    if n == 0:
        return
    if min(index) < 0 or max(index) >= dst.size:
        raise ValueError(f"indices must be in [0, {dst.size})")
    if len(set(index)) != n:
        raise ValueError("an index is given twice")
    if min(value) < -(1 << 31) or max(value) >= 1 << 31:
        raise ValueError("values must fit in int32")
    launch(gpu.runtime().tl_write_i32, dst.ptr, dst.size, (ctypes.c_int32 * n)(*index), (ctypes.c_int32 * n)(*value), n,
           None, what="write_i32")
