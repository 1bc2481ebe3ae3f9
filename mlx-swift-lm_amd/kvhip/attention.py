"""`attentionWithCacheUpdate` (AttentionUtils.swift:37-95) over libkvhip caches."""
from __future__ import annotations

from .cache import BlockScaledKVCache, MaskMode, QuantizedKVCache


def attention_with_cache_update(queries, keys, values, cache, scale, mask=None):
    """Update `cache` with the new keys/values and attend; returns [B,Hq,L,Dv].

    Quantized caches take the `updateQuantized` + `quantizedScaledDotProductAttention`
    branch (AttentionUtils.swift:72-85), others `update` + fused SDPA (:86-93); both
    run as one C-ABI call, kvhip_cache_update_attend.
    """
    if cache is None:
        raise ValueError("a kvhip cache is required; cache-less attention is outside this path")
    return cache.update_attend(queries, keys, values, scale, mask)


def quantized_scaled_dot_product_attention(queries, cache: QuantizedKVCache, scale, mask=None):
    """`quantizedScaledDotProductAttention` (KVCache.swift:2351-2447) over the rows
    `cache` already holds (the quantized tuples stay in device pages)."""
    return cache.attend(queries, scale, mask or MaskMode.none())


def sparse_attention_with_cache_update(queries, keys, values, cache: BlockScaledKVCache, scale, count, first=1, recent=1, left_pad=None):
    """Update `cache` and attend over `count` blocks of 64 positions that each token chooses: [B,Hq,L,Dv].  Runs as one C-ABI
    call, kvhip_cache_update_attend_blocks; no counterpart in the reference."""
    return cache.update_attend_blocks(queries, keys, values, scale, count, first, recent, left_pad)[0]
