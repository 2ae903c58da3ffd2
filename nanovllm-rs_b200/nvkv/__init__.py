"""nvkv: B200 (sm_100a) attention hot path of nanovllm_rs behind its own
operator surface.  Importing this package loads libnvkv.so and fails if it is
missing; there is no CPU or PyTorch fallback."""
from ._lib import NvkvError, device_error, lib, LIB_PATH  # noqa: F401
from .ops import (load_kvcache_fp8b, paged_attention, paged_attention_fp8b,  # noqa: F401
                  qknorm_rope, rope, rope_append, rope_frequencies, store_kvcache, workspace_size,
                  workspace_size_fp8b)
from .layers import (Attention, Context, get_context, reset_context,  # noqa: F401
                     set_context, store_kv_cache)

__all__ = ["Attention", "Context", "NvkvError", "device_error", "get_context",
           "load_kvcache_fp8b", "paged_attention", "paged_attention_fp8b", "qknorm_rope",
           "reset_context", "rope", "rope_append", "rope_frequencies", "set_context",
           "store_kv_cache", "store_kvcache", "workspace_size", "workspace_size_fp8b"]
