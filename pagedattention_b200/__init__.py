"""pagedattention_b200 — B200-native (sm_100a) paged-attention decode.

Drop-in for the decode path of lashhw/pagedattention: the same
``flash_attn_with_kvcache_wrapper_*`` signature (src/common.py:1-14) backed by
hand-written CUDA kernels in ``libpab200.so`` (C ABI: include/pab200.h).
"""
from .common import _validate_decode_inputs
from .int4 import (
    int4_cache,
    int4_page_bytes,
    kv_append_int4,
    kv_read_int4,
    paged_attention_int4,
)
from .kernel_b200 import (
    default_scale,
    flash_attn_with_kvcache_wrapper_b200,
    kv_append,
    kv_append_status,
    merge_packed_states,
    merge_states,
    paged_attention,
    paged_attention_exchange,
    paged_attention_states,
    read_status,
    state_numel,
)
from .sparse import paged_attention_sparse, select_pages, update_page_bounds

__all__ = [
    "_validate_decode_inputs",
    "default_scale",
    "flash_attn_with_kvcache_wrapper_b200",
    "int4_cache",
    "int4_page_bytes",
    "kv_append",
    "kv_append_int4",
    "kv_append_status",
    "kv_read_int4",
    "merge_packed_states",
    "merge_states",
    "paged_attention",
    "paged_attention_exchange",
    "paged_attention_int4",
    "paged_attention_sparse",
    "paged_attention_states",
    "read_status",
    "select_pages",
    "state_numel",
    "update_page_bounds",
]
