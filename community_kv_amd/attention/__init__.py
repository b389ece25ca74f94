"""Attention adapters, cache types, selection, and decode primitives."""

from community_kv_amd.attention.adapter import ATTENTION_IMPLEMENTATION, CommunityKVAttention, HuggingFaceAttention
from community_kv_amd.attention.cache import StaticCache, StaticCacheLayer
from community_kv_amd.attention.decode import DecodeLayerWorkspace, decode_layer
from community_kv_amd.attention.flash_attention import prefill_attention_topk
from community_kv_amd.attention.kernels.packed_segments import PackedSegments
from community_kv_amd.attention.quantized import QuantizedKVCache, evict, quantized_append, quantized_attention
from community_kv_amd.attention.quantized_cache import QuantizedCache, QuantizedCacheAttention, QuantizedCacheLayer

__all__ = [
    "ATTENTION_IMPLEMENTATION",
    "CommunityKVAttention",
    "DecodeLayerWorkspace",
    "HuggingFaceAttention",
    "PackedSegments",
    "QuantizedCache",
    "QuantizedCacheAttention",
    "QuantizedCacheLayer",
    "QuantizedKVCache",
    "StaticCache",
    "StaticCacheLayer",
    "decode_layer",
    "evict",
    "prefill_attention_topk",
    "quantized_append",
    "quantized_attention",
]
