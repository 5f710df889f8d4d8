"""Attention of one new token a sequence where groups of sequences begin with the same pages (additive API).

:func:`~triton_llm.kernels.paged_attention_decode` reads the whole cache of every sequence.  Where sequences begin alike -- a
system prompt, a document, the beams of one search -- and :class:`~triton_llm.paged_cache.PagedKVCache` holds those pages
once, :func:`paged_attention_shared` reads them once too, for all sequences of a group together.

Who shares what is put together once a step by :func:`plan_shared_attention`, on the device, from lengths that only the
device has to know; every layer's call goes by that plan.
"""

from __future__ import annotations

import numpy as np

from triton_llm import _lib, gpu
from ._common import default_scale, launch, scratch
from .paged import _BF16, _check_heads, _check_pool, _check_table, _is_int32, _same_output, check_page_size, dtype_code_of

__all__ = ["SharedPlan", "plan_shared_attention", "paged_attention_shared", "shared_workspace_bytes"]


class SharedPlan:
    """What :func:`plan_shared_attention` leaves on the device, and the sizes that it is for."""

    def __init__(self, sizes, nbytes: int):
        self.sizes = sizes  # (batch, max_pages, n_groups, n_head, n_kv_head, d_k, page_size, dtype code)
        self.buffer = gpu.allocate((nbytes,), np.uint8)


def shared_workspace_bytes(batch: int, n_groups: int, n_head: int, n_kv_head: int, d_k: int) -> int:
    """Bytes of a ``workspace`` for :func:`paged_attention_shared` (0: the sizes are not supported)."""
    return int(_lib.load().tl_shared_workspace_bytes(batch, n_groups, n_head, n_kv_head, d_k))


@gpu.plan_cache(256)
def _plan_sizes(table, lens, members, starts, shared, n_head, n_kv_head, d_k, page_size, code):
    """(sizes, bytes of the plan) of a call by its shapes."""
    check_page_size(page_size)
    batch, max_pages = _check_table(table, lens, None, page_size, 1 << 30)
    _check_heads(n_head, n_kv_head, n_kv_head, d_k)
    if members != (batch,):
        raise ValueError(f"members must be int32 of shape ({batch},), got {members}")
    if len(shared) != 1 or shared[0] < 1 or starts != (shared[0] + 1,):
        raise ValueError(f"shared_lens must be int32 (n_groups,) and group_starts (n_groups + 1,), got {shared} and {starts}")
    sizes = (batch, max_pages, shared[0], n_head, n_kv_head, d_k, page_size, code)
    need = _lib.load().tl_shared_plan_bytes(batch, shared[0], n_head, n_kv_head, d_k)
    if need == 0:
        raise ValueError(f"{batch} sequences in {shared[0]} groups with {n_head} / {n_kv_head} heads are not supported (batch "
                         f"and groups <= 65535, n_head / n_kv_head <= 128)")
    return sizes, need


def plan_shared_attention(page_table, cache_lens, members, group_starts, shared_lens, n_head: int, n_kv_head: int, d_k: int,
                          page_size: int, dtype, len_add: int = 0, plan: SharedPlan | None = None) -> SharedPlan:
    """The plan of a step: group g is the sequences ``members[group_starts[g] : group_starts[g + 1]]``, whose first
    ``shared_lens[g]`` positions lie in the same pages (any number of positions; only the first sequence's entries of the
    table are read for whole blocks of 16 of them).

    page_table: int32 ``(batch, max_pages)``; cache_lens and members: int32 ``(batch,)``; group_starts: int32 ``(n_groups + 1,)``;
    shared_lens: int32 ``(n_groups,)``, all on the device.  Sequence b sees ``cache_lens[b] + len_add`` positions.  A member outside ``[0,
    batch)`` is none; a sequence in no group is not computed, one that is named twice counts where it is named last.  One that is shorter than ``shared_lens[g]``, or the only one
    of its group, shares nothing, and nobody does where a group's start lies below the one before it.  The plan holds for every layer, for as long as lengths, groups and table stay.  ``plan``: an
    earlier plan, which is written over if its sizes fit (it may be in use by calls issued before).
    """
    if not (page_table.dtype.char == cache_lens.dtype.char == members.dtype.char == group_starts.dtype.char
            == shared_lens.dtype.char == "i"):
        for name, t in (("page_table", page_table), ("cache_lens", cache_lens), ("members", members),
                        ("group_starts", group_starts), ("shared_lens", shared_lens)):
            if not _is_int32(t):
                raise ValueError(f"{name} must be int32, got {gpu.dtype_name(t.dtype)} {t.shape}")
    sizes, need = _plan_sizes(page_table.shape, cache_lens.shape, members.shape, group_starts.shape, shared_lens.shape, n_head,
                              n_kv_head, d_k, page_size, _BF16 if dtype is gpu.bfloat16 else gpu.dtype_code(dtype))
    if not -(1 << 31) <= len_add < 1 << 31:
        raise ValueError(f"len_add must fit in int32, got {len_add}")
    if plan is None or plan.sizes != sizes or plan.buffer.nbytes < need:
        plan = SharedPlan(sizes, need)
    launch(gpu.runtime().tl_shared_plan, cache_lens.ptr, int(len_add), members.ptr, group_starts.ptr, shared_lens.ptr, sizes[0],
           sizes[2], n_head, n_kv_head, d_k, sizes[1], page_size, sizes[7], plan.buffer.ptr, plan.buffer.nbytes, None,
           what="plan_shared_attention")
    return plan


@gpu.plan_cache(256)
def _call_plan(pool, v_pool, table, q, sizes, n_head, n_kv_head):
    n_pages, n_kv, page_size, d_k = _check_pool(pool, v_pool)
    batch, max_pages = _check_table(table, None, None, page_size, 1 << 30)
    _check_heads(n_head, n_kv_head, n_kv, d_k)
    if q != (batch, n_head, d_k) and q != (batch, 1, n_head, d_k):
        raise ValueError(f"q shape {q} is not (batch={batch}, n_head={n_head}, d_k={d_k})")
    if sizes[:2] + sizes[3:7] != (batch, max_pages, n_head, n_kv_head, d_k, page_size):
        raise ValueError(f"the plan is for (batch, max_pages, n_head, n_kv_head, d_k, page_size) = {sizes[:2] + sizes[3:7]}, "
                         f"the call for {(batch, max_pages, n_head, n_kv_head, d_k, page_size)}")
    q_str = _lib.strides(n_head * d_k, d_k)
    p_str = _lib.strides(n_kv * page_size * d_k, page_size * d_k, d_k)
    need = _lib.load().tl_shared_workspace_bytes(batch, sizes[2], n_head, n_kv_head, d_k)
    return (max_pages, n_pages, page_size), (batch, n_head, n_kv_head, d_k, q_str, p_str, p_str, q_str), need


def paged_attention_shared(q_dev, k_pages, v_pages, page_table, plan: SharedPlan, n_head: int, n_kv_head: int,
                           sm_scale: float | None = None, out=None, workspace=None):
    """One query per sequence, ``(batch, n_head, d_k)``, over its pages, by a plan of the step.

    Results are those of ``paged_attention_decode`` without a window, to the rounding of sums in
    32 bits.  A sequence that sees nothing gives zeros; the rows of sequences in no group are left
    as they were.  ``out`` overlaps no input.
    """
    if not _is_int32(page_table):
        raise ValueError(f"page_table must be int32, got {gpu.dtype_name(page_table.dtype)} {page_table.shape}")
    pages, dims, need = _call_plan(k_pages.shape, v_pages.shape, page_table.shape, q_dev.shape, plan.sizes, n_head, n_kv_head)
    code = dtype_code_of(q_dev, k_pages, v_pages)
    if code != plan.sizes[7]:
        raise ValueError(f"the plan is for dtype code {plan.sizes[7]}, the call has {code}")
    out = _same_output(out, q_dev)
    ws = scratch(need, workspace, key="shared")
    if sm_scale is None:
        sm_scale = default_scale(dims[3])
    launch(gpu.runtime().tl_paged_attention_shared, q_dev.ptr, k_pages.ptr, v_pages.ptr, page_table.ptr, *pages,
           plan.buffer.ptr, plan.buffer.nbytes, plan.sizes[2], out.ptr, ws.ptr, ws.nbytes, *dims, float(sm_scale), code, None,
           what="paged_attention_shared")
    return out
