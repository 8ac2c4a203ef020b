"""Host checks and planning of decode behind a shared prefix (CPU)."""
import ctypes

import pytest

from inkling_fa4 import _abi

_P = 1 << 20  # fake, aligned device address (never dereferenced)
OK, EINVAL, EUNSUPPORTED, EWORKSPACE = 0, 1, 2, 3


def _call(args=None, kv=None, prefix=None, quant=None, batch=2, ws=None, ws_bytes=0):
    base = dict(batch=batch, n_heads=8, kv_heads=2, head_dim=128, rel_extent=128, rel_width=128,
                max_seqlen_q=1, max_seqlen_k=1024, total_q=batch, total_k=0, q=_P, k=2 * _P,
                v=3 * _P, rel=4 * _P, out=5 * _P, cu_seqlens_q=6 * _P, q_stride_t=1024,
                q_stride_h=128, k_stride_t=256, k_stride_h=128, v_stride_t=256, v_stride_h=128,
                rel_stride_t=1024, rel_stride_h=128, out_stride_t=1024, out_stride_h=128,
                softmax_scale=0.1, qkv_dtype=_abi.IFA4_BF16, rel_dtype=_abi.IFA4_FP32,
                flags=_abi.IFA4_FLAG_BOTTOM_RIGHT)
    a = _abi.make_args(**dict(base, **(args or {})))
    pk = _abi.make_paged(**dict(dict(
        block_size=16, block_table=_P, seqused_k=2 * _P, block_table_stride=64,
        k_stride_block=4096, v_stride_block=4096, num_blocks=100, max_blocks_per_seq=64), **(kv or {})))
    sp = _abi.make_shared_prefix(**dict(dict(prefix_len=512, prefix_table=_P, prefix_blocks=32),
                                        **(prefix or {})))
    q = ctypes.byref(_abi.make_quant(**quant)) if quant is not None else None
    lib = _abi.lib()
    refs = ctypes.byref(a), ctypes.byref(pk), ctypes.byref(sp), q
    return (lib.ifa4_decode_shared_workspace_bytes(*refs),
            lib.ifa4_decode_shared_fwd(*refs, ws, ws_bytes, None))


@pytest.mark.parametrize("kw,want", [
    ({}, EWORKSPACE),  # every check passed: the workspace is asked for
    ({"prefix": {"prefix_len": 0, "prefix_table": 0, "prefix_blocks": 0}}, EWORKSPACE),
    ({"prefix": {"struct_size": 4}}, EINVAL),
    ({"prefix": {"prefix_len": -1}}, EINVAL),
    ({"prefix": {"prefix_len": 513}}, EINVAL),         # more than the table holds
    ({"prefix": {"prefix_table": 0}}, EINVAL),
    ({"prefix": {"prefix_table": _P + 2}}, EINVAL),
    ({"prefix": {"prefix_blocks": -1, "prefix_len": 0}}, EINVAL),
    ({"args": {"flags": 0}}, EUNSUPPORTED),            # top-left
    ({"args": {"total_q": 3}}, EINVAL),
    ({"args": {"n_heads": 64, "kv_heads": 2}}, EUNSUPPORTED),  # a group of 32
    ({"args": {"head_dim": 96}}, EUNSUPPORTED),
    ({"args": {"max_seqlen_k": 1025}}, EINVAL),        # past the table
    ({"args": {"rel_stride_t": 1 << 28}}, EUNSUPPORTED),  # a sequence's bias rows (decode's check)
    # 1999 (4095) strides of 2^18 fp32 values: below (past) 2 GiB of bias
    ({"args": {"rel_stride_t": 1 << 18}, "batch": 2000}, EWORKSPACE),
    ({"args": {"rel_stride_t": 1 << 18}, "batch": 4096}, EUNSUPPORTED),
    ({"args": {"q": _P + 8}}, EUNSUPPORTED),
    ({"kv": {"block_size": 24}}, EINVAL),
    ({"kv": {"block_table": 0}}, EINVAL),
    ({"quant": {"k_scale": 0.0}}, EINVAL),
    ({"quant": {}, "args": {"head_dim": 64, "k_stride_h": 64}, "kv": {"block_size": 8}},
     EUNSUPPORTED),                                    # a wave load of 16 rows in one block
    ({"quant": {}}, EWORKSPACE),
    ({"batch": 0}, OK),
    ({"ws": ctypes.c_void_p(_P), "ws_bytes": 256}, EWORKSPACE),
    ({"ws": ctypes.c_void_p(_P + 16), "ws_bytes": 1 << 30}, EWORKSPACE),
])
def test_checks(kw, want):
    size, status = _call(**kw)
    assert status == want
    assert (size > 0) == (want == EWORKSPACE)


def test_null_arguments():
    lib = _abi.lib()
    a = _abi.make_args()
    assert lib.ifa4_decode_shared_fwd(ctypes.byref(a), None, None, None, None, 0, None) == EINVAL
    assert lib.ifa4_decode_shared_workspace_bytes(None, None, None, None) == 0
