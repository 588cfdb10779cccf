"""Slots, paged keys/values per layer group, and fixed-size per-sequence state."""
from .allocators import CacheError, CacheFull, IndexPool
from .blocks import BlockStore, EvictionPolicy, parse_cache_dtype
from .cache import (PAGE_TOKENS, Cache, CacheRequest, KVGroup, KVLayerView, KVRequest, StateGroup,
                    StateLayerView, StateRequest)

__all__ = ["BlockStore", "EvictionPolicy", "parse_cache_dtype", "CacheError", "CacheFull", "IndexPool", "PAGE_TOKENS", "Cache", "CacheRequest", "KVGroup",
           "KVLayerView", "KVRequest", "StateGroup", "StateLayerView", "StateRequest"]
