"""Page tables that the GPU keeps (additive API).

:class:`~triton_llm.paged_cache.PageTables` deals pages on the host, which has to know every length.
Where the lengths lie on the device -- speculative or captured steps, many steps without the
host -- the tables can be kept there:

* :func:`assign_kv_pages` -- pages for a step's new tokens: table entries, and for every row of the packed batch its slot
  and its position;
* :func:`release_kv_pages` -- the pages of ended sequences back on the free list.

The free list is a stack ``free_pages`` ``(n_pages,)`` int32 with ``counts`` ``(2,)`` int32 beside it, ``counts[0]`` pages on it;
the page taken next is its last.  A packed batch has the sequences' new tokens one behind the other: sequence b's are rows
``starts[b] .. starts[b + 1] - 1``.  Nothing here synchronises or copies to the host, and a captured call
goes by the numbers that are there when it is replayed.

A step: :func:`assign_kv_pages`, then in every layer :func:`~triton_llm.kernels.paged_kv_append_slots` and
:func:`~triton_llm.kernels.paged_attention_packed` (or, for one token of every sequence,
:func:`~triton_llm.kernels.paged_attention_shared`); ``ends`` are the next step's ``cache_lens``.
"""

from __future__ import annotations

import functools

import numpy as np

from triton_llm import _lib, gpu
from ._common import launch, scratch
from .paged import _is_int32, _ptr, check_page_size

__all__ = ["assign_kv_pages", "release_kv_pages", "pages_workspace_bytes"]


def pages_workspace_bytes(batch: int) -> int:
    """Bytes of a ``workspace`` for :func:`assign_kv_pages` (0: such a batch is not supported)."""
    return int(_lib.load().tl_pages_workspace_bytes(batch))


# What a call's shapes allow is found once for each combination of them, as in paged.py; types are looked at in every call.

def _check_int32(**tensors) -> None:
    for name, t in tensors.items():
        if t is not None and not _is_int32(t):
            raise ValueError(f"{name} must be int32, got {gpu.dtype_name(t.dtype)} {t.shape}")


def _check_pages(table, free, page_size, counts, counts_out):
    if len(table) != 2 or min(table) < 1:
        raise ValueError(f"page_table must be int32 (batch, max_pages), got {table}")
    check_page_size(page_size)
    if len(free) != 1 or free[0] < 1:
        raise ValueError(f"free_pages must be int32 (n_pages,), got {free}")
    for shape in (counts, counts_out):
        if shape != (2,):
            raise ValueError(f"counts must be int32 of shape (2,), got {shape}")
    if max(free[0], table[1]) * page_size >= 1 << 31:
        raise ValueError(f"{max(free[0], table[1])} pages of {page_size} exceed 2^31 - 1 positions")
    need = pages_workspace_bytes(table[0])
    if need == 0:
        raise ValueError(f"a batch of {table[0]} is not supported (at most 65535)")
    return need


def _check_vectors(**vectors) -> None:
    for name, (shape, n) in vectors.items():
        if shape is not None and shape != (n,):
            raise ValueError(f"{name} must be int32 of shape ({n},), got {shape}")


@functools.lru_cache(maxsize=256)
def _release_plan(table, free, page_size, counts, counts_out, lens, ended, keep, lens_out):
    _check_pages(table, free, page_size, counts, counts_out)
    n = table[0]
    _check_vectors(lens=(lens, n), ended=(ended, n), keep=(keep, n), lens_out=(lens_out, n))
    return n, table[1], free[0]


@functools.lru_cache(maxsize=256)
def _assign_plan(table, free, page_size, counts, counts_out, cache_lens, new_lens, max_tokens, slots, positions, starts, ends):
    need = _check_pages(table, free, page_size, counts, counts_out)
    n = table[0]
    _check_vectors(cache_lens=(cache_lens, n), new_lens=(new_lens, n), slots=(slots, max_tokens), positions=(positions, max_tokens),
                   starts=(starts, n + 1), ends=(ends, n))
    return n, table[1], free[0], need


def release_kv_pages(page_table, lens, ended, free_pages, counts, page_size: int, keep=None, lens_out=None, counts_out=None):
    """Give the pages of sequences with ``ended[b] != 0`` back; returns ``(lens_out, counts_out)``.

    They are those of columns ``keep[b]`` (int32 ``(batch,)``: leading pages that others have too; None: 0) up to
    ``ceil(lens[b] / page_size)`` of the table, entries that name no page left out, and go behind the free list's last
    by sequence and column.  ``lens_out`` (default: ``lens`` itself) is 0 for an ended sequence and ``lens`` for the others;
    ``counts_out`` (default: ``counts`` itself) the pages on the list and how many had no room on it (none, unless a page is given back twice).
    The table stays as it is.
    """
    if lens_out is None:
        lens_out = lens
    if counts_out is None:
        counts_out = counts
    if not (page_table.dtype.char == lens.dtype.char == ended.dtype.char == free_pages.dtype.char == counts.dtype.char
            == lens_out.dtype.char == counts_out.dtype.char == "i" and (keep is None or keep.dtype.char == "i")):
        _check_int32(page_table=page_table, lens=lens, ended=ended, free_pages=free_pages, counts=counts, keep=keep,
                     lens_out=lens_out, counts_out=counts_out)
    batch, max_pages, n_pages = _release_plan(page_table.shape, free_pages.shape, page_size, counts.shape, counts_out.shape,
                                              lens.shape, ended.shape, None if keep is None else keep.shape, lens_out.shape)
    launch(gpu.runtime().tl_release_pages, page_table.ptr, max_pages, page_size, lens.ptr, ended.ptr, _ptr(keep), batch,
           free_pages.ptr, n_pages, counts.ptr, counts_out.ptr, lens_out.ptr, None, what="release_kv_pages")
    return lens_out, counts_out


def assign_kv_pages(cache_lens, new_lens, page_table, free_pages, counts, page_size: int, max_tokens: int, out=None,
                    counts_out=None, workspace=None):
    """Pages for ``new_lens[b]`` more tokens of each sequence; returns ``(slots, positions, starts, ends)``, int32 on the device.

    Sequences are granted pages in their order: b is, if what it and those before it need is on the free list (or it
    needs none), its tokens fit in its row of the table and its rows below ``max_tokens``.  New pages are written to
    the rows of ``page_table``.  ``slots`` and ``positions`` ``(max_tokens,)``: ``page * page_size + row`` and the position of every row of
    the packed batch, -1 for rows of a sequence that was not granted and behind the last; ``starts`` ``(batch + 1,)``: each
    sequence's first row, also of one that was not granted: :func:`~triton_llm.kernels.paged_attention_packed` goes by ``starts``
    alone, so what it leaves in rows of slot -1 holds nothing of meaning (their keys were not written, and a row of ``page_table`` that was released
    still names pages that others may hold) and is to be dropped.  ``ends`` ``(batch,)``: ``cache_lens`` and what was granted.  ``counts_out`` (default: ``counts`` itself):
    pages left, and the sequences with new tokens that were not granted.  ``out``: the four tensors, which
    overlap no input.
    """
    if counts_out is None:
        counts_out = counts
    if not 0 <= max_tokens < 1 << 31:
        raise ValueError(f"max_tokens must be >= 0 and fit in int32, got {max_tokens}")
    if out is None:
        batch = page_table.shape[0] if page_table.shape else 0
        out = tuple(gpu.allocate((n,), np.int32) for n in (max_tokens, max_tokens, batch + 1, batch))
    elif len(out) != 4:
        raise ValueError(f"out must be (slots, positions, starts, ends), got {len(out)} tensors")
    slots, positions, starts, ends = out
    if not (cache_lens.dtype.char == new_lens.dtype.char == page_table.dtype.char == free_pages.dtype.char == counts.dtype.char
            == counts_out.dtype.char == slots.dtype.char == positions.dtype.char == starts.dtype.char == ends.dtype.char == "i"):
        _check_int32(cache_lens=cache_lens, new_lens=new_lens, page_table=page_table, free_pages=free_pages, counts=counts,
                     slots=slots, positions=positions, starts=starts, ends=ends, counts_out=counts_out)
    batch, max_pages, n_pages, need = _assign_plan(page_table.shape, free_pages.shape, page_size, counts.shape, counts_out.shape,
                                                   cache_lens.shape, new_lens.shape, max_tokens, slots.shape, positions.shape,
                                                   starts.shape, ends.shape)
    ws = scratch(need, workspace, key="pages")
    launch(gpu.runtime().tl_assign_pages, cache_lens.ptr, new_lens.ptr, batch, page_table.ptr, max_pages, page_size,
           free_pages.ptr, n_pages, counts.ptr, counts_out.ptr, max_tokens, slots.ptr, positions.ptr, starts.ptr, ends.ptr,
           ws.ptr, ws.nbytes, None, what="assign_kv_pages")
    return out
