"""Inkling relative-position-bias flash attention, MI355X (gfx950) native.

Same export names as the reference package (src/inkling_fa4/__init__.py:1-11),
minus `ref_rel_attn`: the fp32 oracle is test infrastructure and lives in the
repository's `oracle/` package, outside the product.  Added: prefill over a paged KV
cache, `inkling_fa4_rel_attention_paged`; the paged-KV
decode entry points `inkling_fa4_rel_attention_decode_paged` and
`inkling_fa4_rel_attention_decode_shared_prefix`; the fused
relative-logit projection `inkling_fa4_rel_attention_rproj`; and the steps before
the attention, `inkling_fa4_qk_norm_rope` and `inkling_fa4_kv_append_paged`; and attention
over chosen blocks of a long cache, `inkling_fa4_key_bounds_paged`,
`inkling_fa4_select_blocks_paged` and `inkling_fa4_rel_attention_sparse_paged`.
"""
from . import autotune_configs
from .norm_rope import inkling_fa4_kv_append_paged, inkling_fa4_qk_norm_rope
from .ops import (
    inkling_fa4_rel_attention,
    inkling_fa4_rel_attention_decode,
    inkling_fa4_rel_attention_decode_paged,
    inkling_fa4_rel_attention_decode_shared_prefix,
    inkling_fa4_rel_attention_decode_triton,
    inkling_fa4_rel_attention_kv_pruned_triton,
    inkling_fa4_rel_attention_paged,
    inkling_fa4_rel_attention_rproj,
    inkling_fa4_rel_attention_triton,
    prefill_tile_counts,
)
from .sparse import (
    inkling_fa4_key_bounds_paged,
    inkling_fa4_rel_attention_sparse_paged,
    inkling_fa4_select_blocks_paged,
)

__all__ = [
    "inkling_fa4_rel_attention",
    "inkling_fa4_rel_attention_decode",
    "inkling_fa4_rel_attention_decode_paged",
    "inkling_fa4_rel_attention_decode_shared_prefix",
    "inkling_fa4_rel_attention_paged",
    "inkling_fa4_rel_attention_triton",
    "inkling_fa4_rel_attention_decode_triton",
    "inkling_fa4_rel_attention_kv_pruned_triton",
    "inkling_fa4_rel_attention_rproj",
    "inkling_fa4_key_bounds_paged",
    "inkling_fa4_select_blocks_paged",
    "inkling_fa4_rel_attention_sparse_paged",
    "inkling_fa4_qk_norm_rope",
    "inkling_fa4_kv_append_paged",
    "prefill_tile_counts",
    "autotune_configs",
]
