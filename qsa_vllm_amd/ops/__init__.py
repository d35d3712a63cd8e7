"""gfx950 HIP operators of the QSA sparse-attention path (reference ``yulan_qsa_vllm/ops``)."""

from .indexer import (decode_select_attend, qsa_select_paged_decode, qsa_select_paged_prefill,
                      select_paged_tokens)
from .int4 import Int4Weight, int4_linear, int4_pack, int4_quantize
from .kv_cache import Int4KVCache, qk_norm_rope, rotary_table
from .logits import LogitsRules, process_logits
from .normalization import IndexerRMSNorm, indexer_norm_rope, rotary_cache
from .paged import qsa_int4_paged_attention, qsa_window_paged_attention
from .prepare import qsa_prepare
from .qsa import (expand_qsa_block_indices_cuda, qsa_compress_groups_with_ratio,
                  qsa_select_paged_tokens, qsa_sparse_paged_attention, qsa_store_cache_rows)
from .topk import topk, topk_expand
from .tree import qsa_tree_paged_attention, tree_ancestors

__all__ = [
    "IndexerRMSNorm",
    "Int4KVCache",
    "Int4Weight",
    "LogitsRules",
    "decode_select_attend",
    "expand_qsa_block_indices_cuda",
    "qsa_compress_groups_with_ratio",
    "qsa_store_cache_rows",
    "indexer_norm_rope",
    "int4_linear",
    "int4_pack",
    "int4_quantize",
    "process_logits",
    "qk_norm_rope",
    "qsa_int4_paged_attention",
    "qsa_prepare",
    "qsa_select_paged_decode",
    "qsa_select_paged_prefill",
    "qsa_select_paged_tokens",
    "qsa_sparse_paged_attention",
    "qsa_tree_paged_attention",
    "qsa_window_paged_attention",
    "rotary_cache",
    "rotary_table",
    "select_paged_tokens",
    "topk",
    "topk_expand",
    "tree_ancestors",
]
