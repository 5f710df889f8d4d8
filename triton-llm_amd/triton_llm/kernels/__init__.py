"""Attention-path kernels of triton_llm on the gfx950 HIP library.

Exports the reference's hot-path names (triton_llm/kernels/__init__.py:6-31 of
ziliangpeng/triton-llm: ``attention``, ``attention_gqa``, ``precompute_cos_sin``,
``apply_rope``) plus the additive batched entry points of this build
(flash prefill, KV-cache append, split-K decode) and the model step's other
layers: the projection ``gemm``, ``rms_norm`` (plus the fused
``add_rms_norm``), ``swiglu`` and ``add``, and on-device next-token
``sample`` / ``sample_rows`` (the models' ``_sample``).  Serving many sequences
adds the cache in pages (append, attention, page copies), attention through a
sliding window, and beam search's selection.  The reference's gelu,
layer_norm, softmax and embedding kernels (GPT-2 and host-side pieces) are
outside this library's scope.
"""

from .attention import attention
from .attention_gqa import attention_gqa
from .rope import apply_rope, precompute_cos_sin, precompute_cos_sin_device
from .flash import flash_attention, flash_attention_strided
from .gemm import gemm, gemm_grouped
from .rms_norm import add_rms_norm, rms_norm
from .swiglu import swiglu
from .add import add
from .sample import sample, sample_rows
from .decode import (
    allocate_kv_cache,
    attention_decode,
    decode_step,
    decode_workspace,
    rope_kv_append,
)
from .paged import (
    allocate_kv_pages,
    copy_kv_pages,
    paged_attention_decode,
    paged_attention_prefill,
    paged_decode_workspace,
    paged_kv_append,
    paged_prefill_workspace_bytes,
    write_i32,
)
from .window import window_attention, window_attention_strided, window_workspace_bytes
from .beam import beam_select, beam_workspace_bytes

__all__ = [
    "attention",
    "attention_gqa",
    "precompute_cos_sin",
    "precompute_cos_sin_device",
    "apply_rope",
    "flash_attention",
    "flash_attention_strided",
    "allocate_kv_cache",
    "rope_kv_append",
    "attention_decode",
    "decode_step",
    "decode_workspace",
    "gemm",
    "gemm_grouped",
    "rms_norm",
    "add_rms_norm",
    "swiglu",
    "add",
    "sample",
    "sample_rows",
    "allocate_kv_pages",
    "paged_kv_append",
    "paged_attention_decode",
    "paged_decode_workspace",
    "paged_attention_prefill",
    "paged_prefill_workspace_bytes",
    "copy_kv_pages",
    "write_i32",
    "window_attention",
    "window_attention_strided",
    "window_workspace_bytes",
    "beam_select",
    "beam_workspace_bytes",
]
