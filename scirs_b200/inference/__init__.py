"""Inference: paged KV cache with shared pages, paged decode and shared-prefix
attention, speculative decoding, and cached generation for the GPT engine."""
from .kv_cache import (BlockManager, BlockManagerConfig, InferenceError, KvPageConfig, KvPagePool, SharedPrefixCache,
                       copy_pages)
from .paged_attention import (PagedAttentionConfig, PagedAttentionForward, paged_attention_reference,
                              shared_prefix_attention_reference)
from .generate import GPTGenerator
from .speculative import (DraftVerification, SpeculativeConfig, SpeculativeDecoder, SpeculativeResult, TokenDist,
                          Xorshift64, verify_drafts)

__all__ = [
    "GPTGenerator",
    "BlockManager", "BlockManagerConfig", "InferenceError", "KvPageConfig", "KvPagePool", "SharedPrefixCache",
    "copy_pages",
    "PagedAttentionConfig", "PagedAttentionForward", "paged_attention_reference",
    "shared_prefix_attention_reference",
    "DraftVerification", "SpeculativeConfig", "SpeculativeDecoder", "SpeculativeResult", "TokenDist", "Xorshift64",
    "verify_drafts",
]
