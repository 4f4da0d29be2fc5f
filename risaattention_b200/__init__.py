"""B200-native RISA quantised attention: the reference package's public names
(src/risa_attention/__init__.py:17-31) over hand-written sm_100a kernels."""
from ._backend import is_available as int8_attention_is_available
from .attention import (PrequantizedInt8Attention, RetainedMassPattern,
                        build_retained_mass_pattern, construct_sparse_int8_attention,
                        construct_sparse_int8_attention_from_prequantized, int8_attention,
                        int8_attention_from_prequantized, is_available, measure_pattern_recall,
                        prequantize_int8_attention, sparse_int8_attention)
from .host_pipeline import int8_attention_from_host
from .permutation import KVPermutation, prepare_kv_permutation
from .serving import (Compaction, Eviction, KeyValueCache, RotaryTable, allocate_key_value_cache, append_to_cache,
                      cached_key_weights, compact_cache, evict_from_cache, fork_sequences, paged_attention,
                      read_from_cache, resize_sequences, rotary_frequencies, rotary_table, rotate_positions)

__all__ = [
    "KVPermutation", "prepare_kv_permutation", "PrequantizedInt8Attention", "RetainedMassPattern",
    "build_retained_mass_pattern", "construct_sparse_int8_attention",
    "construct_sparse_int8_attention_from_prequantized", "int8_attention",
    "int8_attention_from_host", "int8_attention_from_prequantized", "int8_attention_is_available", "measure_pattern_recall",
    "prequantize_int8_attention", "sparse_int8_attention", "Eviction", "KeyValueCache", "RotaryTable",
    "allocate_key_value_cache", "append_to_cache", "cached_key_weights", "evict_from_cache",
    "Compaction", "compact_cache", "fork_sequences", "resize_sequences",
    "paged_attention", "read_from_cache", "rotary_frequencies", "rotary_table", "rotate_positions",
]
__version__ = "0.1.0"
