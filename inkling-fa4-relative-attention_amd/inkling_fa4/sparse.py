"""Attention over some blocks of a long paged cache: which blocks a token reads, and the
attention over them.

The reference has none of it; its serving caller keeps a paged cache
(outputs/architecture.md:117-120), and every decode step reads all of it.  A step here is

    inkling_fa4_kv_append_paged(...)                       # new keys and values
    inkling_fa4_key_bounds_paged(k_cache, bounds, ...)     # bounds of the blocks they went to
    blocks = inkling_fa4_select_blocks_paged(q, bounds, ...)
    out = inkling_fa4_rel_attention_sparse_paged(q, k_cache, v_cache, rel, ..., blocks, ...)

for one new token a sequence or a chunk of a prompt alike.  cu_seqlens_q, seqused_k (which
counts the new tokens) and block_table are the append's and the paged attention's throughout;
what they and the lists hold never leads to an access outside the tensors.
"""
from .ops import _call, _op, _resolve, _window_left


def inkling_fa4_key_bounds_paged(k_cache, bounds, cu_seqlens_q, seqused_k, block_table,
                                 max_seqlen_q):
    """Least and greatest key element, by kv head and dimension, of the blocks that new tokens
    went to: bounds [num_blocks, Hkv, 2, D] in k_cache's dtype (bf16, fp16 or float8_e4m3fn) changes
    in place, bounds[block, h, 0] the minimum over the block's keys below seqused_k, [.., 1] the
    maximum (exact; NaN where a key is NaN).  Other blocks keep theirs.  The blocks are read
    whole, so a block given to another sequence needs nothing but this call after its append.
    Where two sequences share a block they fill to unequal lengths, each bound is that of either.

    max_seqlen_q must bound the new tokens of a sequence.  There is no derivative: tangents are
    refused, and so are bounds that require a gradient (outside torch.no_grad()).
    """
    _op("key_bounds_paged")(k_cache, bounds, cu_seqlens_q, seqused_k, block_table,
                            int(max_seqlen_q))


def inkling_fa4_select_blocks_paged(q, bounds, cu_seqlens_q, seqused_k, block_table, block_size,
                                    max_seqlen_q, max_seqlen_k, n_select, *, sink_blocks=1,
                                    recent_blocks=2):
    """The blocks that each token and kv head attends to: int32 [total_q, Hkv, n_select],
    ascending, then -1 (a token of no sequence: -1 throughout).

    Token i of a sequence's n sits at position p = seqused_k[b] - n + i and may read blocks
    0 .. p // block_size.  Where they are more than n_select, it reads the first sink_blocks,
    the last recent_blocks (at least one, its own), and the best of the others by
        score = sum over the kv head's query heads g and d of max(q_gd lo_d, q_gd hi_d),
    an upper bound of the sum over those heads of q . k for any key of the block (the relative
    bias has no part in it: recent_blocks covers what it favours), from q [total_q, Hq, D] (bf16,
    fp16) and bounds as inkling_fa4_key_bounds_paged leaves them (of q's dtype or float8_e4m3fn).
    Scores are summed in 64 bits: only those closer than such a sum's rounding may rank either
    way from one batch to another; equal bounds score equal, and equal scores go to the lower
    block.  A score of NaN counts as infinity, and so does a block with an infinite or NaN bound.
    max_seqlen_q and max_seqlen_k must bound the lengths.

    Where max_seqlen_k has more than n_select blocks, the call holds a score of 8 bytes for every
    token, kv head and block of max_seqlen_k: 8 * total_q * Hkv * ceil(max_seqlen_k / block_size)
    bytes from torch's allocator (512 MiB for 4096 tokens, 2 heads and 128K keys in blocks of 16).
    Take long chunks over long caches in parts, and give a tight max_seqlen_k.  A step that mixes a
    chunk with single tokens is faster as two calls, one for each kind.
    """
    return _call("select_blocks_paged", q, bounds, cu_seqlens_q, seqused_k, block_table,
                 int(block_size), int(max_seqlen_q), int(max_seqlen_k), int(n_select),
                 int(sink_blocks), int(recent_blocks))


def inkling_fa4_rel_attention_sparse_paged(q, k_cache, v_cache, rel_logits, cu_seqlens_q,
                                           seqused_k, block_table, blocks, max_seqlen_q,
                                           max_seqlen_k, rel_extent, window_size=(-1, -1), *,
                                           softmax_scale=None, return_lse=False, k_scale=1.0,
                                           v_scale=1.0):
    """inkling_fa4_rel_attention_paged (causal) over the blocks that each token and kv head
    lists: blocks int32 [total_q, Hkv, n_select], as inkling_fa4_select_blocks_paged gives them
    or any other way.  An entry that is no block of the sequence (-1), lies past the token, or
    whose table entry lies outside the pool is passed over; a block named twice counts twice.
    A token whose list holds no visible key: out 0, lse -inf; rows of tokens that no sequence
    holds are not written.  What a token does not see may hold anything, infinities and NaN too.

    The bias and the window go by the keys' positions in the sequence, listed or not.  GQA groups
    up to 16; caches, types and the other arguments as in inkling_fa4_rel_attention_paged; no
    gradient either.
    """
    if k_cache.dim() != 4:
        raise ValueError("k_cache must be [num_blocks, block_size, kv_heads, head_dim]")
    scale = _resolve(q, k_cache.shape[1:], None, None, None, softmax_scale)
    out, lse = _call("sparse_paged", q, k_cache, v_cache, rel_logits, cu_seqlens_q, seqused_k,
                     block_table, blocks, int(max_seqlen_q), int(max_seqlen_k), int(rel_extent),
                     _window_left(window_size), scale, bool(return_lse), float(k_scale),
                     float(v_scale))
    return (out, lse) if return_lse else out
