"""The steps between the projections and the attention: RMS norm of query and key
heads with the position rotation in one pass, and the same on the way into a paged
KV cache.

The reference has neither as a kernel; its serving caller norms the heads before the
attention and writes a paged cache (outputs/architecture.md:24-50,117-127).

Formulas, per head row x [head_dim] of a token at position p, in fp32 with one rounding
to the input's dtype at the end:
    z = x / sqrt(mean(x^2) + eps) * weight         (weight None: z = x)
    y = z, its rot_dim leading elements turned by the angles of p: the pair (a, b) with
        angle i becomes (a cos[p, i] - b sin[p, i], b cos[p, i] + a sin[p, i]);
        pairs are elements i and i + rot_dim / 2, or 2 i and 2 i + 1 (interleaved=True)
rot_dim is twice the columns of cos and sin (a multiple of 16, at most head_dim);
cos=None: no rotation.  head_dim 64 or 128, bf16 or fp16.  Contents of positions,
cu_seqlens, seqused_k and block tables stay on the device and are not checked against
the contract; what they hold never leads to an access outside the tensors.
"""
from ._native import ops as _ops

_overloads = {}


def _op(name):
    op = _overloads.get(name)
    if op is None:
        op = _overloads[name] = getattr(_ops(), name).default
    return op


def inkling_fa4_qk_norm_rope(q, k, q_weight=None, k_weight=None, cos=None, sin=None,
                             positions=None, *, eps=1e-6, interleaved=False):
    """RMS norm of every query and key head and the rotation by the token's position.

    q [tokens, Hq, D], k [tokens, Hkv, D] (bf16 or fp16, last dim contiguous, rows 16-byte
    aligned: column ranges of one projection's output are fine), q_weight / k_weight [D]
    (bf16, fp16 or fp32, both of one dtype) or None, cos / sin [positions, rot_dim / 2] fp32
    or None, positions int32 [tokens] (needed with cos; outside the table: results
    unspecified).  Returns (q, k), contiguous, in the inputs' dtype.

    Differentiable in q, k and the weights (once, in reverse mode; tangents are refused);
    the backward pass reads the inputs again and keeps nothing else.  The weights' gradients
    are summed over tokens and heads in fp32, in a fixed order.
    """
    if q_weight is None and k_weight is None and cos is None:
        raise ValueError("nothing to do: give a weight, or cos and sin")
    return _op("qk_norm_rope")(q, k, q_weight, k_weight, cos, sin, positions, float(eps),
                               bool(interleaved))


def inkling_fa4_kv_append_paged(k, v, k_cache, v_cache, cu_seqlens_q, seqused_k, block_table, *,
                                q=None, q_weight=None, k_weight=None, cos=None, sin=None,
                                eps=1e-6, interleaved=False, k_scale=1.0, v_scale=1.0):
    """Write new keys and values into a paged KV cache, k normed and turned on the way.

    k, v [tokens, Hkv, D] are the new tokens of all sequences one after the other
    (cu_seqlens_q int32 [batch + 1]); k_cache / v_cache [num_blocks, block_size, Hkv, D],
    block_table int32 [batch, max_blocks] and seqused_k int32 [batch] are what
    inkling_fa4_rel_attention_decode_paged takes afterwards: seqused_k counts the new keys,
    so token i of n new ones has position p = seqused_k[b] - n + i and goes to row
    p % block_size of block block_table[b, p // block_size].  The caches change in place;
    rows that no token goes to stay as they are.  cos and sin need a row for every position
    p (a token past them gets unspecified values).

    With q [tokens, Hq, D] the queries are normed and turned by the same positions in the
    same launch and returned (else None); rows of tokens that no sequence holds are not
    written.  A float8_e4m3fn cache stores the e4m3 values nearest to the fp32 quotients
    k / k_scale and v / v_scale (ties to even, saturating; a 16-bit cache ignores the
    scales).  A token with p < 0, past the table or whose table entry lies outside the pool
    is not written; two tokens sent to one row leave one of the two.

    There is no gradient: the result never requires one, tangents are refused, and so are
    caches that require a gradient (outside torch.no_grad()).
    """
    out = _op("kv_append_paged")(k, v, k_cache, v_cache, cu_seqlens_q, seqused_k, block_table, q,
                                 q_weight, k_weight, cos, sin, float(eps), bool(interleaved),
                                 float(k_scale), float(v_scale))
    return out if q is not None else None
