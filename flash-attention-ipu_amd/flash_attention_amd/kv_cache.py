"""A block cache of 8-bit keys and values and causal attention over it: what a generation loop needs beside `flash_attention_qkv_packed`.

    cache_tables             block tables, positions and slots of a step, from the requests' lengths, on the device
    cache_append             a step's keys and values into the cache: e4m3 codes, one scale per block of tokens and head
    flash_attention_cached   attention of single tokens, drafts and prompts of ragged requests over the cache
    KVCache                  the tensors of a model's layers and the calls above in the order of a step
"""

from ._impl.kv_cache import BLOCK_SIZES, CacheStep, KVCache, cache_append, cache_tables, cache_width, flash_attention_cached

__all__ = ["BLOCK_SIZES", "CacheStep", "KVCache", "cache_append", "cache_tables", "cache_width", "flash_attention_cached"]
