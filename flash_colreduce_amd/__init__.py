"""MI355X-native attention column reduction (same package surface as the reference:
flash_colreduce/__init__.py:1-4)."""
from .cache import KVCache, cache_keep, cache_read, cache_write, chunk_attention, tree_attention
from .drafts import PagePool, Verified, cache_accept, cache_reserve, verify_drafts
from .flash import flash_colreduce, flash_colreduce_multi, row_lse2, topk_keep_mask
from .naive import naive_colreduce

__version__ = "0.1.0"
__all__ = ["flash_colreduce", "flash_colreduce_multi", "naive_colreduce", "row_lse2", "topk_keep_mask",
           "KVCache", "cache_write", "cache_read", "cache_keep", "tree_attention", "chunk_attention",
           "Verified", "verify_drafts", "cache_accept", "PagePool", "cache_reserve", "__version__"]
