"""B200-native paged-KV attention path with the call surface of lite_llama's
``kv_engine`` / paged-attention modules.

* :mod:`.kernels` — ``update_kv_buffer``, ``flash_decoding``,
  ``paged_chunk_flash_attention``, ``flash_attention2_no_pad`` (CUDA, via libb200kv.so), and the same
  over a 4-bit cache (``*_kv4``)
* :mod:`.paged_attention` — ``PagedKVCacheManager``, ``PagedReqTokensManager``
* :mod:`.kv_engine` — refcounts, prefix cache, prefill packer and chunk planner
"""

from .kv_engine import (  # noqa: F401
    ChunkedPrefillPlanner,
    KVBlockRefCounter,
    MixedLengthPrefillPacker,
    PackedPrefillPlan,
    PackedPrefillRequest,
    PrefillChunk,
    PrefixCache,
    PrefixCacheMatch,
)
from .paged_attention import PagedKVCacheManager, PagedReqTokensManager  # noqa: F401
from .kernels import (  # noqa: F401
    empty_kv4_buffer,
    flash_attention2_no_pad,
    flash_decoding,
    flash_decoding_kv4,
    fused_qk_norm_rope_append_kv4,
    gather_kv_buffer_kv4,
    paged_chunk_flash_attention,
    paged_chunk_flash_attention_kv4,
    update_kv_buffer,
    update_kv_buffer_kv4,
    update_kv_buffer_kv4_split,
    update_kv_buffer_split,
)

__version__ = "0.1.0"
