"""CPU tests of the C ABI of the paged prefill, the key bounds, the block choice and the attention
over listed blocks: what is refused before a launch, and workspaces.  Addresses are made up: no
check reads them, and no accepted call here gets as far as a launch."""
import ctypes
import math

import pytest

from inkling_fa4 import _abi

OK, EINVAL, EUNSUPPORTED, EWORKSPACE = 0, _abi.IFA4_EINVAL, _abi.IFA4_EUNSUPPORTED, _abi.IFA4_EWORKSPACE
P = 1 << 20
BR = _abi.IFA4_FLAG_BOTTOM_RIGHT


def args(**kw):
    base = dict(flags=BR, q=P, k=P, v=P, rel=P, out=P, cu_seqlens_q=P, q_stride_t=1024,
                q_stride_h=128, k_stride_t=256, k_stride_h=128, v_stride_t=256, v_stride_h=128,
                rel_stride_t=1024, rel_stride_h=128, out_stride_t=1024, out_stride_h=128, total_q=64,
                batch=4, n_heads=8, kv_heads=2, head_dim=128, rel_extent=128, rel_width=128,
                max_seqlen_q=16, max_seqlen_k=8000, softmax_scale=0.1, qkv_dtype=_abi.IFA4_BF16,
                rel_dtype=_abi.IFA4_BF16)
    return _abi.make_args(**dict(base, **kw))


def paged(**kw):
    base = dict(block_size=16, block_table=P, seqused_k=P, block_table_stride=512,
                k_stride_block=4096, v_stride_block=4096, num_blocks=2000, max_blocks_per_seq=512)
    return _abi.make_paged(**dict(base, **kw))


def lists(**kw):
    return _abi.make_block_list(**dict(dict(n_select=64, blocks=P, stride_t=128, stride_h=64), **kw))


def ref(x):
    return None if x is None else ctypes.byref(x)


def prefill(a, kv, qt=None, ws=None, n=0):
    return _abi.lib().ifa4_prefill_paged_fwd(ref(a), ref(kv), ref(qt), ws, n, None)


def sparse(a, kv, ls, qt=None, ws=None, n=0):
    return _abi.lib().ifa4_sparse_paged_fwd(ref(a), ref(kv), ref(ls), ref(qt), ws, n, None)


BAD_ATTENTION = [
    (dict(flags=0), {}, EUNSUPPORTED), (dict(head_dim=96), {}, EUNSUPPORTED),
    (dict(n_heads=7), {}, EINVAL), (dict(softmax_scale=math.nan), {}, EINVAL),
    (dict(softmax_scale=-1.0), {}, EUNSUPPORTED), (dict(q=0), {}, EINVAL), (dict(k=0), {}, EINVAL),
    (dict(rel=0), {}, EINVAL), (dict(rel_extent=129), {}, EINVAL), (dict(k=P + 8), {}, EUNSUPPORTED),
    (dict(k_stride_t=260), {}, EUNSUPPORTED), (dict(max_seqlen_k=8193), {}, EINVAL),
    (dict(cu_seqlens_q=0), {}, EINVAL), ({}, dict(block_size=24), EINVAL),
    ({}, dict(block_size=4), EINVAL), ({}, dict(struct_size=8), EINVAL),
    ({}, dict(block_table=0), EINVAL), ({}, dict(seqused_k=2), EINVAL), ({}, dict(num_blocks=0), EINVAL),
    ({}, dict(k_stride_block=4100), EUNSUPPORTED),
    ({}, dict(max_blocks_per_seq=(1 << 26) + 1), EUNSUPPORTED),
]


@pytest.mark.parametrize("a,kv,want", BAD_ATTENTION)
def test_attention_refusals(a, kv, want):
    assert prefill(args(**a), paged(**kv)) == want
    assert sparse(args(**a), paged(**kv), lists()) == want
    lib = _abi.lib()
    assert lib.ifa4_prefill_paged_workspace_bytes(ref(args(**a)), ref(paged(**kv)), None) == 0
    assert lib.ifa4_sparse_paged_workspace_bytes(ref(args(**a)), ref(paged(**kv)), ref(lists()), None) == 0


def test_attention_refusals_of_missing_structs_and_scales():
    assert prefill(None, paged()) == EINVAL and prefill(args(), None) == EINVAL
    assert sparse(args(), paged(), None) == EINVAL
    for kw in (dict(k_scale=0.0), dict(v_scale=math.inf), dict(struct_size=4)):
        assert prefill(args(), paged(), _abi.make_quant(**kw)) == EINVAL
        assert sparse(args(), paged(), lists(), _abi.make_quant(**kw)) == EINVAL
    quant = _abi.make_quant()
    # one load covers 16 rows of 64 bytes, which one block has to hold
    small = dict(head_dim=64, q_stride_h=64, k_stride_h=64, v_stride_h=64, out_stride_h=64)
    assert prefill(args(**small), paged(block_size=8, max_blocks_per_seq=1024), quant) == EUNSUPPORTED


@pytest.mark.parametrize("ls,want", [(dict(n_select=0), EINVAL), (dict(blocks=0), EINVAL),
                                     (dict(blocks=P + 2), EINVAL), (dict(stride_t=-1), EINVAL),
                                     (dict(struct_size=0), EINVAL), (dict(n_select=1 << 27), EUNSUPPORTED)])
def test_list_refusals(ls, want):
    assert sparse(args(), paged(), lists(**ls)) == want


def test_sparse_refusals():
    assert sparse(args(causal=0), paged(), lists()) == EUNSUPPORTED
    wide = dict(n_heads=34, kv_heads=2, q_stride_t=4352, out_stride_t=4352)
    assert sparse(args(**wide), paged(), lists()) == EUNSUPPORTED  # GQA groups up to 16
    assert sparse(args(total_q=1 << 26), paged(), lists()) == EUNSUPPORTED


def test_attention_workspaces():
    lib = _abi.lib()
    a, kv = args(), paged()
    n = lib.ifa4_prefill_paged_workspace_bytes(ref(a), ref(kv), None)
    assert n > 0 and n % 256 == 0  # few tiles over long caches: split
    assert prefill(a, kv) == EWORKSPACE and prefill(a, kv, ws=P, n=n - 1) == EWORKSPACE
    assert prefill(a, kv, ws=P + 16, n=n) == EWORKSPACE
    n = lib.ifa4_sparse_paged_workspace_bytes(ref(a), ref(kv), ref(lists()), None)
    assert n > 0 and n % 256 == 0
    assert sparse(a, kv, lists()) == EWORKSPACE and sparse(a, kv, lists(), ws=P, n=n - 1) == EWORKSPACE
    many = args(total_q=4096, max_seqlen_q=2000)
    assert lib.ifa4_sparse_paged_workspace_bytes(ref(many), ref(kv), ref(lists()), None) == 0


def test_nothing_to_do():
    for kw in (dict(batch=0), dict(max_seqlen_q=0), dict(total_q=0, q=0, out=0, rel=0)):
        assert prefill(args(**kw), paged()) == OK
        assert sparse(args(**kw), paged(), lists()) == OK


def bounds(kv=None, **kw):
    base = dict(kv_dtype=_abi.IFA4_BF16, head_dim=128, kv_heads=2, batch=4, max_seqlen_q=16, k_cache=P,
                k_stride_t=256, k_stride_h=128, bounds=P, bounds_stride_block=512, bounds_stride_h=256,
                cu_seqlens=P)
    return _abi.lib().ifa4_key_bounds_paged(ref(_abi.make_key_bounds(**dict(base, **kw))),
                                            ref(kv if kv is not None else paged()), None)


@pytest.mark.parametrize("kw,want", [
    (dict(struct_size=4), EINVAL), (dict(kv_dtype=_abi.IFA4_FP32), EUNSUPPORTED),
    (dict(head_dim=96), EUNSUPPORTED), (dict(head_dim=0), EINVAL), (dict(kv_heads=0), EINVAL),
    (dict(batch=-1), EINVAL), (dict(max_seqlen_q=-1), EINVAL), (dict(k_cache=0), EINVAL),
    (dict(k_cache=P + 8), EUNSUPPORTED), (dict(k_stride_t=252), EUNSUPPORTED), (dict(bounds=0), EINVAL),
    (dict(bounds=P + 4), EUNSUPPORTED), (dict(bounds_stride_h=128), EUNSUPPORTED),
    (dict(bounds_stride_block=0), EUNSUPPORTED), (dict(cu_seqlens=0), EINVAL),
    (dict(batch=70000), EUNSUPPORTED)])
def test_bounds_refusals(kw, want):
    assert bounds(**kw) == want


def test_bounds_table_refusals_and_nothing_to_do():
    assert bounds(paged(block_size=24)) == EINVAL and bounds(paged(num_blocks=0)) == EINVAL
    assert bounds(paged(struct_size=1)) == EINVAL and bounds(paged(block_table=0)) == EINVAL
    assert bounds(paged(max_blocks_per_seq=1 << 27)) == EUNSUPPORTED
    assert bounds(batch=0) == OK and bounds(max_seqlen_q=0) == OK


def select_args(**kw):
    base = dict(dtype=_abi.IFA4_BF16, kv_dtype=_abi.IFA4_BF16, head_dim=128, n_heads=8, kv_heads=2,
                batch=4, max_seqlen_q=16, max_seqlen_k=8000, n_select=64, sink_blocks=1,
                recent_blocks=2, total_q=64, q=P, q_stride_t=1024, q_stride_h=128, bounds=P,
                bounds_stride_block=512, bounds_stride_h=256, cu_seqlens=P, blocks=P)
    return _abi.make_block_select(**dict(base, **kw))


def select(kv=None, ws=None, n=0, **kw):
    return _abi.lib().ifa4_select_blocks_paged(
        ref(select_args(**kw)), ref(kv if kv is not None else paged()), ws, n, None)


@pytest.mark.parametrize("kw,want", [
    (dict(struct_size=4), EINVAL), (dict(dtype=_abi.IFA4_FP32), EUNSUPPORTED),
    (dict(kv_dtype=_abi.IFA4_FP16), EUNSUPPORTED), (dict(head_dim=32), EUNSUPPORTED),
    (dict(n_heads=7), EINVAL), (dict(kv_heads=0), EINVAL), (dict(n_select=0), EINVAL),
    (dict(sink_blocks=-1), EINVAL), (dict(recent_blocks=0), EINVAL), (dict(sink_blocks=63), EINVAL),
    (dict(max_seqlen_k=8193), EINVAL), (dict(total_q=-1), EINVAL), (dict(q=0), EINVAL),
    (dict(q=P + 8), EUNSUPPORTED), (dict(q_stride_h=100), EUNSUPPORTED), (dict(bounds=0), EINVAL),
    (dict(bounds_stride_block=4), EUNSUPPORTED), (dict(blocks=0), EINVAL), (dict(cu_seqlens=3), EINVAL),
    (dict(batch=70000), EUNSUPPORTED), (dict(total_q=1 << 26), EUNSUPPORTED)])
def test_select_refusals(kw, want):
    assert select(**kw) == want
    assert _abi.lib().ifa4_select_blocks_workspace_bytes(ref(select_args(**kw)), ref(paged())) == 0


def test_select_workspace_and_nothing_to_do():
    lib = _abi.lib()
    n = lib.ifa4_select_blocks_workspace_bytes(ref(select_args()), ref(paged()))
    assert n > 0 and n % 256 == 0
    assert select() == EWORKSPACE and select(ws=P, n=n - 1) == EWORKSPACE
    assert select(ws=P + 8, n=n) == EWORKSPACE
    # every list holds all blocks: no scores
    assert lib.ifa4_select_blocks_workspace_bytes(ref(select_args(n_select=500)), ref(paged())) == 0
    # nor where no sequence has a token
    for kw in (dict(batch=0), dict(max_seqlen_q=0)):
        assert lib.ifa4_select_blocks_workspace_bytes(ref(select_args(**kw)), ref(paged())) == 0
    assert select(total_q=0) == OK and select(total_q=0, blocks=0, q=0) == OK


def test_grids_of_less_than_2_to_the_32_threads():
    """More workgroups than a launch holds are refused before it."""
    wide = dict(kv_heads=1 << 12, n_heads=1 << 12, q_stride_t=1 << 19)
    assert select(paged(max_blocks_per_seq=1 << 20), total_q=1, max_seqlen_q=1, max_seqlen_k=1 << 24,
                  **wide) == EUNSUPPORTED
    assert select(total_q=1 << 23) == EUNSUPPORTED
    assert bounds(paged(max_blocks_per_seq=1 << 24), max_seqlen_q=1 << 28) == EUNSUPPORTED
    assert sparse(args(total_q=(1 << 25) - 4), paged(), lists()) == EUNSUPPORTED
