"""Beam search's selection on the HIP library (additive API).

The reference samples one sequence (smollm2_triton/model.py:566-584, here
:mod:`~triton_llm.kernels.sample`); :func:`beam_select` keeps the best
continuations of several: every ``(beam, token)`` of a batch item scored
``scores[b, j] + log_softmax(logits[b, j])[token]``, the ``n_select`` best of them
returned best first.  The sequences' states follow their parents by a change of page tables
(:meth:`triton_llm.paged_cache.PagedKVCache.reorder`).
"""

from __future__ import annotations

import functools
import math

import numpy as np

from triton_llm import _lib, gpu
from ._common import launch, scratch

__all__ = ["beam_select", "beam_workspace_bytes", "max_select"]


def max_select() -> int:
    """Most continuations a call selects per batch item."""
    return int(_lib.load().tl_beam_max_select())


def beam_workspace_bytes(batch: int, beams: int, vocab: int) -> int:
    """Bytes of a ``workspace`` for :func:`beam_select` (0: the sizes are not supported)."""
    return int(_lib.load().tl_beam_select_workspace_bytes(batch, beams, vocab))


@functools.lru_cache(maxsize=256)
def _plan(scores, logits, n_select):
    """(batch, beams, vocab, n_select, workspace bytes) of a call by its shapes."""
    if len(scores) != 2:
        raise ValueError(f"scores must be float32 (batch, beams), got {scores}")
    batch, beams = scores
    if len(logits) < 2 or logits[-1] <= 0:
        raise ValueError(f"logits must be (batch * beams, vocab) with vocab > 0, got {logits}")
    vocab = logits[-1]
    if math.prod(logits[:-1]) != batch * beams:
        raise ValueError(f"logits {logits} do not hold {batch} x {beams} rows")
    n_select = 2 * beams if n_select is None else int(n_select)
    if n_select < 0:
        raise ValueError(f"n_select must be >= 0, got {n_select}")
    need = 0
    if batch and n_select:
        lib = _lib.load()
        need = lib.tl_beam_select_workspace_bytes(batch, beams, vocab)
        if need == 0 or n_select > lib.tl_beam_max_select():
            raise ValueError(f"selecting {n_select} of {batch} x {beams} rows of vocab {vocab} is not supported "
                             f"(n_select <= {lib.tl_beam_max_select()}, beams <= 64, batch * beams <= 65535, "
                             f"vocab <= 262144)")
    return batch, beams, vocab, n_select, need


def beam_select(logits_dev, scores_dev, n_select: int | None = None, out=None, workspace=None):
    """(scores, parents, tokens), each ``(batch, n_select)`` on the device: float32, int32, int32.

    logits_dev: ``(batch * beams, vocab)`` or ``(batch, beams, vocab)`` in a compute
    dtype; scores_dev: ``(batch, beams)`` float32.  n_select: default ``2 * beams`` (room for
    beams that end).  Scores are ordered in 64 bits (the softmax's logarithm
    to 2^-44); ties go to the lowest
    ``beam * vocab + token``.  A beam whose score is not finite, or whose logits hold NaN,
    +inf or nothing but -inf, has no continuations, and a logit of -inf is none;
    where fewer are left the rest are ``(-inf, -1, -1)``.  No synchronisation.
    """
    if scores_dev.dtype.char != "f":
        raise ValueError(f"scores must be float32 (batch, beams), got {gpu.dtype_name(scores_dev.dtype)}")
    code = gpu.dtype_code(logits_dev.dtype)
    batch, beams, vocab, n_select, need = _plan(scores_dev.shape, logits_dev.shape, n_select)
    shape = (batch, n_select)
    if out is None:
        out = tuple(gpu.allocate(shape, t) for t in (np.float32, np.int32, np.int32))
    elif len(out) != 3 or any(o.shape != shape or o.dtype.char != c for o, c in zip(out, "fii")):
        raise ValueError(f"out must be float32, int32 and int32 tensors of shape {shape}")
    if batch == 0 or n_select == 0:
        return out
    ws = scratch(need, workspace, key="beam")
    launch(gpu.runtime().tl_beam_select, logits_dev.ptr, scores_dev.ptr, batch, beams, vocab, vocab, n_select,
           out[0].ptr, out[1].ptr, out[2].ptr, ws.ptr, ws.nbytes, code, None, what="beam_select")
    return out
