"""Causal attention through a sliding window with sinks (additive API).

``window_attention`` is :func:`~triton_llm.kernels.flash.flash_attention` with a
bounded view: a query at position p sees the keys ``p - window < j <= p`` and the first
``sinks`` keys of the sequence; ``window = 0`` sees every ``j <= p``.  Positions are
bottom-right aligned, query i at ``seq_k - seq_q + i`` (attention_gqa.py:97 of the
reference, which has no windows); a query before position 0 sees nothing and gives
zeros.  Keys outside of every row's view are not read.

:func:`~triton_llm.kernels.paged.paged_attention_prefill` is the same over a cache in pages.
"""

from __future__ import annotations

import functools

from triton_llm import _lib, gpu
from ._common import contiguous_strides, default_scale, launch, scratch
from .paged import check_window, dtype_code_of


@gpu.plan_cache(1024)
def _strided_plan(batch, n_head, n_kv_head, seq_q, seq_k, d_k, q_strides, k_strides, v_strides, o_strides, window, sinks):
    """The C entry's sizes and strides in their order, and its workspace's bytes by dtype code."""
    if n_head <= 0 or n_kv_head <= 0 or n_head % n_kv_head:
        raise ValueError(f"n_head ({n_head}) must be a positive multiple of n_kv_head ({n_kv_head})")
    if d_k not in (64, 128):
        raise ValueError(f"window attention supports d_k in (64, 128), got {d_k}")
    check_window(window, sinks)
    sizes = (batch, n_head, n_kv_head, seq_q, seq_k, d_k, _lib.strides(*q_strides), _lib.strides(*k_strides),
             _lib.strides(*v_strides), _lib.strides(*o_strides))
    ws = [_lib.load().tl_window_workspace_bytes(batch, n_head, n_kv_head, seq_q, seq_k, d_k, window, sinks, code)
          for code in range(3)] if batch and seq_q and seq_k else None
    return sizes, ws


def window_workspace_bytes(batch: int, n_head: int, n_kv_head: int, seq_q: int, seq_k: int, d_k: int, dtype, window: int = 0,
                           sinks: int = 0) -> int:
    """Bytes of a ``workspace`` for a call with these sizes (0: none is used)."""
    check_window(window, sinks)
    return _lib.load().tl_window_workspace_bytes(batch, n_head, n_kv_head, seq_q, seq_k, d_k, window, sinks,
                                                 gpu.dtype_code(dtype))


def window_attention_strided(q, k, v, out, *, batch, n_head, n_kv_head, seq_q, seq_k, d_k, q_strides, k_strides,
                             v_strides, o_strides, window, sinks=0, sm_scale=None, workspace=None):
    """The kernel on raw layouts given by {batch, head, seq} element strides."""
    sizes, ws_bytes = _strided_plan(batch, n_head, n_kv_head, seq_q, seq_k, d_k, tuple(q_strides), tuple(k_strides),
                                    tuple(v_strides), tuple(o_strides), window, sinks)
    code = dtype_code_of(q, k, v, out)
    if batch == 0 or seq_q == 0:
        return out
    if seq_k == 0:
        raise ValueError("seq_k must be >= 1")
    if sm_scale is None:
        sm_scale = default_scale(d_k)
    ws = scratch(ws_bytes[code], workspace, key="window")
    launch(gpu.runtime().tl_window_attention, q.ptr, k.ptr, v.ptr, out.ptr, None if ws is None else ws.ptr,
           0 if ws is None else ws.nbytes, *sizes, float(sm_scale), int(window), int(sinks), code, None,
           what="window_attention")
    return out


@functools.lru_cache(maxsize=1024)
def _contiguous(q, k, v):
    """The arguments of :func:`window_attention_strided` for contiguous tensors of these shapes."""
    if len(q) != 4 or len(k) != 4 or k != v:
        raise ValueError(f"expected q (B,Hq,Sq,D) and k/v (B,Hkv,Sk,D), got {q}, {k}, {v}")
    batch, n_head, seq_q, d_k = q
    kb, n_kv, seq_k, kd = k
    if kb != batch or kd != d_k:
        raise ValueError(f"q {q} and k {k} disagree on batch or d_k")
    qs, ks = contiguous_strides(q)[:3], contiguous_strides(k)[:3]
    return dict(batch=batch, n_head=n_head, n_kv_head=n_kv, seq_q=seq_q, seq_k=seq_k, d_k=d_k, q_strides=qs,
                k_strides=ks, v_strides=ks, o_strides=qs)


def window_attention(q, k, v, window: int, sinks: int = 0, sm_scale: float | None = None, out=None, workspace=None):
    """q ``(batch, n_head, seq_q, d_k)``, k/v ``(batch, n_kv_head, seq_k, d_k)``, contiguous; returns out like q."""
    layout = _contiguous(q.shape, k.shape, v.shape)
    if out is None:
        out = gpu.allocate(q.shape, q.dtype)
    elif out.shape != q.shape:
        raise ValueError(f"out shape {out.shape} != q shape {q.shape}")
    return window_attention_strided(q, k, v, out, **layout, window=window, sinks=sinks, sm_scale=sm_scale,
                                    workspace=workspace)
