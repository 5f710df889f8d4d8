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
import math

import numpy as np

from triton_llm import _lib, gpu
from ._common import default_scale, launch, same_dtype, scratch, vp

MIN_PAGE, MAX_PAGE = 16, 1024


def _check_page_size(page_size: int) -> None:
    if not (MIN_PAGE <= page_size <= MAX_PAGE and page_size & (page_size - 1) == 0):
        raise ValueError(f"page_size must be a power of 2 in [{MIN_PAGE}, {MAX_PAGE}], got {page_size}")


def allocate_kv_pages(n_pages: int, n_kv_head: int, page_size: int, d_k: int, dtype=np.float32, zero: bool = True):
    """(k_pages, v_pages), each ``(n_pages, n_kv_head, page_size, d_k)`` on the GPU."""
    if n_pages <= 0 or n_kv_head <= 0 or d_k <= 0:
        raise ValueError(f"pool dims must be positive, got n_pages={n_pages} n_kv_head={n_kv_head} d_k={d_k}")
    _check_page_size(page_size)
    gpu.dtype_code(dtype)
    alloc = gpu.zeros if zero else gpu.allocate
    shape = (n_pages, n_kv_head, page_size, d_k)
    return alloc(shape, dtype), alloc(shape, dtype)


def _check_pool(k_pages, v_pages):
    if len(k_pages.shape) != 4 or k_pages.shape != v_pages.shape:
        raise ValueError(f"k_pages/v_pages must be matching 4-D (n_pages, n_kv_head, page_size, d_k), "
                         f"got {k_pages.shape} and {v_pages.shape}")
    if min(k_pages.shape) <= 0:
        raise ValueError(f"pool dims must be positive, got {k_pages.shape}")
    _check_page_size(k_pages.shape[2])
    return k_pages.shape


def _check_table(page_table, cache_lens, page_size, most):
    if gpu.dtype_name(page_table.dtype) != "int32" or len(page_table.shape) != 2 or page_table.shape[1] < 1:
        raise ValueError(f"page_table must be int32 (batch, max_pages), got {gpu.dtype_name(page_table.dtype)} "
                         f"{page_table.shape}")
    batch, max_pages = page_table.shape
    if max_pages * page_size > most:
        raise ValueError(f"{max_pages} pages of {page_size} exceed {most} positions")
    _check_lens("cache_lens", cache_lens, batch)
    return batch, max_pages


def _check_lens(name, lens, batch):
    if gpu.dtype_name(lens.dtype) != "int32" or tuple(lens.shape) != (batch,):
        raise ValueError(f"{name} must be int32 of shape ({batch},), got {gpu.dtype_name(lens.dtype)} {lens.shape}")


def _check_heads(n_head, n_kv_head, n_kv, d_k):
    if n_kv != n_kv_head:
        raise ValueError(f"pool has {n_kv} KV heads, n_kv_head={n_kv_head}")
    if n_head <= 0 or n_head % n_kv_head:
        raise ValueError(f"n_head ({n_head}) must be a positive multiple of n_kv_head ({n_kv_head})")
    if d_k not in (64, 128):
        raise ValueError(f"paged attention supports d_k in (64, 128), got {d_k}")


def check_window(window: int, sinks: int) -> None:
    if not (0 <= window < 1 << 31 and 0 <= sinks < 1 << 31):
        raise ValueError(f"window and sinks must be >= 0 and fit in int32, got {window} and {sinks}")


def _same_output(out, q):
    if out is None:
        return gpu.allocate(q.shape, q.dtype)
    if tuple(out.shape) != tuple(q.shape) or gpu.dtype_name(out.dtype) != gpu.dtype_name(q.dtype):
        raise ValueError(f"out must be like q, {q.shape} {gpu.dtype_name(q.dtype)}, got {out.shape} "
                         f"{gpu.dtype_name(out.dtype)}")
    return out


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
    n_pages, n_kv, page_size, d_k = _check_pool(k_pages, v_pages)
    batch, max_pages = _check_table(page_table, cache_lens, page_size, (1 << 31) - 1)
    if len(k_new.shape) not in (3, 4):
        raise ValueError(f"k_new must be 3-D or 4-D, got {k_new.shape}")
    n_new = 1 if len(k_new.shape) == 3 else k_new.shape[1]
    want = (batch, n_kv, d_k) if len(k_new.shape) == 3 else (batch, n_new, n_kv, d_k)
    if tuple(k_new.shape) != want:
        raise ValueError(f"k_new shape {k_new.shape} is not {want} (table {page_table.shape}, pool {k_pages.shape})")
    if tuple(v_new.shape) != want:
        raise ValueError(f"v_new shape {v_new.shape} != k_new shape {k_new.shape}")
    if d_k % 2:
        raise ValueError(f"d_k must be even, got {d_k}")
    n_head = 0
    if q_dev is not None:
        if len(q_dev.shape) != len(want) or q_dev.shape[:-2] != want[:-2] or q_dev.shape[-1] != d_k:
            raise ValueError(f"q shape {q_dev.shape} does not match k_new {k_new.shape}")
        n_head = q_dev.shape[-2]
        if n_head <= 0 or n_head % n_kv:
            raise ValueError(f"n_head ({n_head}) must be a positive multiple of n_kv_head ({n_kv})")
        q_out = q_dev if q_out is None else _same_output(q_out, q_dev)
    elif q_out is not None:
        raise ValueError("q_out is given without q_dev")
    tensors = [k_new, v_new, k_pages, v_pages] + ([q_dev, q_out] if q_dev is not None else [])
    code = same_dtype(*tensors)
    if new_lens is not None:
        _check_lens("new_lens", new_lens, batch)
    if (cos_dev is None) != (sin_dev is None):
        raise ValueError("cos_dev and sin_dev must both be given or both be None")
    rows = rotary = 0
    if cos_dev is not None:
        if (cos_dev.shape != sin_dev.shape or len(cos_dev.shape) != 2 or not 1 <= cos_dev.shape[1] <= d_k // 2
                or cos_dev.dtype != np.float32 or sin_dev.dtype != np.float32):
            raise ValueError(f"cos/sin tables must be float32 (rows, r // 2) with r <= {d_k}, got {cos_dev.shape} "
                             f"and {sin_dev.shape}")
        rows, rotary = cos_dev.shape[0], 2 * cos_dev.shape[1]
    q_str = _lib.strides(n_new * n_head * d_k, n_head * d_k, d_k)
    kv_str = _lib.strides(n_new * n_kv * d_k, n_kv * d_k, d_k)
    p_str = _lib.strides(n_kv * page_size * d_k, page_size * d_k, d_k)
    launch(gpu.runtime().tl_paged_kv_append, vp(q_dev), vp(q_out), vp(k_new), vp(v_new), vp(k_pages), vp(v_pages),
           vp(page_table), max_pages, n_pages, page_size, vp(cache_lens), vp(new_lens), vp(cos_dev), vp(sin_dev),
           rows, rotary, 1 if interleaved else 0, batch, n_new, n_head, n_kv, d_k, q_str, q_str, kv_str, kv_str,
           p_str, p_str, code, None, what="paged_kv_append")
    return q_out


def paged_decode_workspace(batch: int, n_head: int, n_kv_head: int, max_ctx: int, d_k: int):
    """A workspace of :func:`paged_attention_decode`, reusable by consecutive calls on the
    library stream (calls that overlap in time need one each).  Its size goes by the heads alone."""
    if n_head <= 0 or n_kv_head <= 0 or n_head % n_kv_head:
        raise ValueError(f"n_head ({n_head}) must be a positive multiple of n_kv_head ({n_kv_head})")
    return gpu.allocate((gpu.runtime().tl_paged_decode_workspace_bytes(n_head, n_kv_head, d_k),), np.uint8)


def paged_attention_decode(q_dev, k_pages, v_pages, page_table, cache_lens, n_head: int, n_kv_head: int,
                           sm_scale: float | None = None, len_add: int = 0, window: int = 0, sinks: int = 0,
                           out=None, workspace=None):
    """One query per sequence, ``(batch, n_head, d_k)``, over ``cache_lens[b] + len_add`` positions.

    Query head h reads KV head ``h // (n_head // n_kv_head)``.  A sequence without
    visible positions gives zeros.  Hidden positions are not read.
    """
    n_pages, n_kv, page_size, d_k = _check_pool(k_pages, v_pages)
    batch, max_pages = _check_table(page_table, cache_lens, page_size, (1 << 31) - 1)
    _check_heads(n_head, n_kv_head, n_kv, d_k)
    check_window(window, sinks)
    if math.prod(q_dev.shape) != batch * n_head * d_k:
        raise ValueError(f"q shape {q_dev.shape} is not (batch={batch}, n_head={n_head}, d_k={d_k})")
    code = same_dtype(q_dev, k_pages, v_pages)
    out = _same_output(out, q_dev)
    if sm_scale is None:
        sm_scale = default_scale(d_k)
    lib = gpu.runtime()
    ws = scratch(lib.tl_paged_decode_workspace_bytes(n_head, n_kv_head, d_k), workspace, key="paged_decode")
    qo = _lib.strides(n_head * d_k, d_k)
    p_str = _lib.strides(n_kv * page_size * d_k, page_size * d_k, d_k)
    launch(lib.tl_paged_attention_decode, vp(q_dev), vp(k_pages), vp(v_pages), vp(page_table), max_pages, n_pages,
           page_size, vp(cache_lens), int(len_add), int(window), int(sinks), vp(out), vp(ws), ws.nbytes, batch,
           n_head, n_kv_head, d_k, qo, p_str, p_str, qo, float(sm_scale), code, None, what="paged_attention_decode")
    return out


def paged_attention_prefill(q_dev, k_pages, v_pages, page_table, cache_lens, n_head: int, n_kv_head: int,
                            new_lens=None, sm_scale: float | None = None, window: int = 0, sinks: int = 0, out=None):
    """Queries ``(batch, n_new, n_head, d_k)`` at positions ``cache_lens[b] + i`` over the pages.

    The new tokens' own k and v are appended before.  ``new_lens`` as in :func:`paged_kv_append`: rows
    behind a sequence's tokens are left as they were.
    """
    n_pages, n_kv, page_size, d_k = _check_pool(k_pages, v_pages)
    batch, max_pages = _check_table(page_table, cache_lens, page_size, 1 << 30)
    _check_heads(n_head, n_kv_head, n_kv, d_k)
    check_window(window, sinks)
    if len(q_dev.shape) != 4 or q_dev.shape[0] != batch or tuple(q_dev.shape[2:]) != (n_head, d_k):
        raise ValueError(f"q shape {q_dev.shape} is not (batch={batch}, n_new, n_head={n_head}, d_k={d_k})")
    n_new = q_dev.shape[1]
    code = same_dtype(q_dev, k_pages, v_pages)
    if new_lens is not None:
        _check_lens("new_lens", new_lens, batch)
    out = _same_output(out, q_dev)
    if sm_scale is None:
        sm_scale = default_scale(d_k)
    q_str = _lib.strides(n_new * n_head * d_k, d_k, n_head * d_k)  # {batch, head, seq}
    p_str = _lib.strides(n_kv * page_size * d_k, page_size * d_k, d_k)
    launch(gpu.runtime().tl_paged_attention_prefill, vp(q_dev), vp(k_pages), vp(v_pages), vp(page_table), max_pages,
           n_pages, page_size, vp(cache_lens), vp(new_lens), vp(out), batch, n_new, n_head, n_kv_head, d_k, q_str,
           p_str, p_str, q_str, float(sm_scale), int(window), int(sinks), code, None, what="paged_attention_prefill")
    return out


def copy_kv_pages(caches, src, dst) -> None:
    """Page ``dst[i]`` = page ``src[i]`` in every pool of ``caches``.

    caches: pools ``(n_pages, n_kv_head, page_size, d_k)`` of one shape and dtype (the K and V
    of every layer).  src / dst: page numbers on the host; no page may be a destination
    twice, or source and destination.  The numbers travel with the launch: nothing
    synchronises, and a captured graph replays the same copies.
    """
    caches = list(caches)
    src, dst = (np.asarray(list(x), dtype=np.int64) for x in (src, dst))
    if src.shape != dst.shape:
        raise ValueError(f"{src.size} source pages, {dst.size} destinations")
    if not caches or src.size == 0:
        return
    shape, dtype = tuple(caches[0].shape), gpu.dtype_name(caches[0].dtype)
    if len(shape) != 4 or min(shape) <= 0:
        raise ValueError(f"pools must be 4-D (n_pages, n_kv_head, page_size, d_k), got {shape}")
    _check_page_size(shape[2])
    for c in caches:
        if tuple(c.shape) != shape or gpu.dtype_name(c.dtype) != dtype:
            raise ValueError(f"pools differ: {shape} {dtype} and {c.shape} {gpu.dtype_name(c.dtype)}")
    if min(src.min(), dst.min()) < 0 or max(src.max(), dst.max()) >= shape[0]:
        raise ValueError(f"page numbers must be in [0, {shape[0]})")
    if np.unique(dst).size != dst.size:
        raise ValueError("a page is a destination twice")
    if np.intersect1d(src, dst).size:
        raise ValueError("a page is source and destination")
    page_bytes = math.prod(shape[1:]) * caches[0].dtype.itemsize
    bases = (ctypes.c_void_p * len(caches))(*[c.data_ptr() for c in caches])
    pairs = [(ctypes.c_int32 * src.size)(*x.tolist()) for x in (src, dst)]
    launch(gpu.runtime().tl_copy_pages, bases, len(caches), page_bytes, page_bytes, shape[0], *pairs, src.size, None,
           what="copy_kv_pages")


def write_i32(dst, index, value) -> None:
    """``dst.flat[index[i]] = value[i]`` for a device int32 tensor, the values on the host: no
    upload, no synchronisation (page table entries, lengths).  Indices must be distinct."""
    if gpu.dtype_name(dst.dtype) != "int32":
        raise ValueError(f"dst must be int32, got {gpu.dtype_name(dst.dtype)}")
    index, value = (np.asarray(x, dtype=np.int64).ravel() for x in (index, value))
    if index.size != value.size:
        raise ValueError(f"{index.size} indices, {value.size} values")
    if index.size == 0:
        return
    if index.min() < 0 or index.max() >= dst.size:
        raise ValueError(f"indices must be in [0, {dst.size})")
    if np.unique(index).size != index.size:
        raise ValueError("an index is given twice")
    if value.min() < -(1 << 31) or value.max() >= 1 << 31:
        raise ValueError("values must fit in int32")
    pairs = [(ctypes.c_int32 * index.size)(*x.tolist()) for x in (index, value)]
    launch(gpu.runtime().tl_write_i32, vp(dst), dst.size, *pairs, index.size, None, what="write_i32")
