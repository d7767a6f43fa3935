"""Kernel-facing helper ops (reference: nkipy/src/nkipy/core/tensor_apis.py:5-24).

``softmax`` and ``rms_norm`` are traced as the NumPy compositions the row
kernels match (a last-axis softmax lowers to the fused softmax launch).
``conv2d`` / ``conv3d`` are exported for import compatibility; this
single-GPU backend has no implementation for them and calling one raises
``NotImplementedError`` naming the backend.

``rotary_append``, ``paged_attention``, ``window_attention`` and ``sample``
are this backend's own: the steps of a serving loop (a paged key / value
cache, attention with a sliding window, the draw of the next token).  Their
contracts stand with their NumPy forms in :mod:`nkipy_amd.core.ops.serving`.
``rotary_append_fp8`` and ``paged_attention_fp8`` keep that cache in 8 bits
(:mod:`nkipy_amd.core.ops.serving_fp8`); ``assign_pages``, ``beam_select`` and
``beam_reorder`` lay out its block tables and run a beam search over it
(:mod:`nkipy_amd.core.ops.beams`).
"""

from nkipy_amd.core.ops import (  # noqa: F401
    assign_pages, beam_reorder, beam_select, constant, conv2d, conv3d, full, full_like, ones_like, paged_attention,
    paged_attention_fp8, rms_norm, rotary_append, rotary_append_fp8, sample, softmax, topk, window_attention, zeros,
    zeros_like,
)

__all__ = [
    "constant",
    "topk",
    "rms_norm",
    "softmax",
    "conv2d",
    "conv3d",
    "zeros",
    "full",
    "rotary_append",
    "paged_attention",
    "window_attention",
    "sample",
    "rotary_append_fp8",
    "paged_attention_fp8",
    "assign_pages",
    "beam_select",
    "beam_reorder",
]
