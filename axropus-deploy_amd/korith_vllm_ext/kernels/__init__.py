"""Decode-attention kernels of the AMF path (reference: korith_vllm_ext/kernels/__init__.py)."""

from __future__ import annotations

from .dispatch import (
    KERNEL_DISPATCH,
    dense_attention,
    int4_sym_attention,
    dispatch_kernel,
    fallback_fp16_kernel,
    get_current_sm_version,
    hip_decode_attention,
    paged_int4_decode,
    register_kernel,
    try_load_cuda_extension,
)
from .paged import (
    SlotMaps,
    build_slot_maps,
    page_key_bounds,
    paged_decode_attention,
    select_pages,
)
from .rows import paged_attention
from .step import (
    Rotary,
    int4_page_pool,
    read_kv_cache,
    rotary_embedding,
    rotary_frequencies,
    write_kv_cache,
)

__all__ = [
    "KERNEL_DISPATCH",
    "Rotary",
    "SlotMaps",
    "build_slot_maps",
    "dense_attention",
    "int4_page_pool",
    "int4_sym_attention",
    "dispatch_kernel",
    "fallback_fp16_kernel",
    "get_current_sm_version",
    "hip_decode_attention",
    "page_key_bounds",
    "paged_attention",
    "paged_decode_attention",
    "paged_int4_decode",
    "read_kv_cache",
    "register_kernel",
    "rotary_embedding",
    "rotary_frequencies",
    "select_pages",
    "try_load_cuda_extension",
    "write_kv_cache",
]
