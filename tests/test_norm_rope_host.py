"""Host checks of the head norm, its backward pass and the paged append (CPU): every refused
argument returns its status before any device call; Python entry points raise."""
import ctypes

import pytest
import torch

from inkling_fa4 import _abi, inkling_fa4_kv_append_paged, inkling_fa4_qk_norm_rope

_P = 1 << 20  # fake, aligned device address (never dereferenced)
OK, EINVAL, EUNSUPPORTED, EWORKSPACE = 0, 1, 2, 3


def _args(**kw):
    base = dict(dtype=_abi.IFA4_BF16, w_dtype=_abi.IFA4_FP32, head_dim=128, n_heads=8, kv_heads=2,
                rot_dim=128, max_position=64, total=0, q=_P, k=2 * _P, q_out=3 * _P, k_out=4 * _P,
                q_stride_t=1024, q_stride_h=128, k_stride_t=256, k_stride_h=128,
                q_out_stride_t=1024, q_out_stride_h=128, k_out_stride_t=256, k_out_stride_h=128,
                q_weight=5 * _P, k_weight=6 * _P, cos=7 * _P, sin=8 * _P, angle_stride=64,
                positions=9 * _P)
    return _abi.make_norm_rope(**dict(base, **kw))


# Without tokens nothing is launched, so a call that passes its checks returns IFA4_OK here;
# refusals that need tokens come before the launch.
SHARED = [
    ({}, OK),
    ({"struct_size": 8}, EINVAL),
    ({"head_dim": 96}, EINVAL),  # rot_dim 128 of 96
    ({"head_dim": 96, "rot_dim": 96}, EUNSUPPORTED),
    ({"head_dim": 0}, EINVAL),
    ({"dtype": _abi.IFA4_FP32}, EUNSUPPORTED),
    ({"dtype": 9}, EINVAL),
    ({"w_dtype": 9}, EINVAL),
    ({"w_dtype": 9, "q_weight": 0, "k_weight": 0}, OK),
    ({"total": -1}, EINVAL),
    ({"total": 1 << 31}, EUNSUPPORTED),
    ({"eps": -1.0}, EINVAL),
    ({"eps": float("nan")}, EINVAL),
    ({"rot_dim": 24}, EUNSUPPORTED),
    ({"rot_dim": 144}, EINVAL),
    ({"rot_dim": -16}, EINVAL),
    ({"cos": 0}, EINVAL),
    ({"sin": 7 * _P + 4}, EUNSUPPORTED),
    ({"max_position": 0}, EINVAL),
    ({"angle_stride": 60}, EINVAL),
    ({"angle_stride": 66}, EUNSUPPORTED),
    ({"rot_dim": 0, "cos": 0, "sin": 0, "max_position": 0, "angle_stride": 0}, OK),
    ({"interleaved": 2}, EINVAL),
    ({"n_heads": -1}, EINVAL),
    ({"q_weight": 5 * _P + 2}, EINVAL),
    ({"q_stride_t": -8}, EINVAL),
    ({"total": 4, "q": 0}, EINVAL),
    ({"total": 4, "q": _P + 8}, EUNSUPPORTED),
    ({"total": 4, "k_stride_h": 4}, EUNSUPPORTED),
]


def _fwd(a):
    return _abi.lib().ifa4_qk_norm_rope_fwd(ctypes.byref(a), None)


@pytest.mark.parametrize("kw,want", SHARED + [
    ({"n_heads": 0}, EINVAL),
    ({"kv_heads": 0}, EINVAL),
    ({"total": 4, "positions": 0}, EINVAL),
    ({"total": 4, "positions": 9 * _P + 2}, EINVAL),
    ({"total": 4, "q_out": 0}, EINVAL),
    ({"total": 4, "q_out_stride_h": 64}, EUNSUPPORTED),  # rows written over one another
    ({"total": 4, "k_out_stride_t": 0}, EUNSUPPORTED),
])
def test_forward_checks(kw, want):
    assert _fwd(_args(**kw)) == want


def test_null_arguments():
    lib = _abi.lib()
    assert lib.ifa4_qk_norm_rope_fwd(None, None) == EINVAL
    assert lib.ifa4_qk_norm_rope_bwd(ctypes.byref(_args()), None, None, 0, None) == EINVAL
    assert lib.ifa4_kv_append_paged(ctypes.byref(_args()), None, None, None) == EINVAL
    assert lib.ifa4_qk_norm_rope_bwd_workspace_bytes(None) == 0


def _grad(**kw):
    base = dict(gq=_P, gk=2 * _P, dq=3 * _P, dk=4 * _P, gq_stride_t=1024, gq_stride_h=128,
                gk_stride_t=256, gk_stride_h=128, dq_stride_t=1024, dq_stride_h=128,
                dk_stride_t=256, dk_stride_h=128, dq_weight=5 * _P, dk_weight=6 * _P)
    return _abi.make_norm_rope_grad(**dict(base, **kw))


@pytest.mark.parametrize("kw,grad,want", [
    ({}, {"dq_weight": 0, "dk_weight": 0}, OK),        # no tokens: nothing to write
    ({}, {}, EINVAL),                                  # ... and no sum to take
    ({"total": 4}, {"struct_size": 8}, EINVAL),
    ({"total": 4}, {}, EWORKSPACE),
    ({"total": 4}, {"dq_weight": 0}, EINVAL),          # a weight without its gradient
    ({"total": 4, "q_weight": 0}, {}, EINVAL),         # a gradient without its weight
    ({"total": 4}, {"gq": 0}, EINVAL),                 # ... without the output's gradient
    ({"total": 4}, {"gq": 0, "gk": 0}, EINVAL),
    ({"total": 4}, {"gq": 0, "gk": 0, "dq_weight": 0, "dk_weight": 0}, OK),
    ({"total": 4}, {"dq": 0}, EINVAL),
    ({"total": 4}, {"gk": 2 * _P + 8}, EUNSUPPORTED),
    ({"total": 4}, {"dk_stride_h": 0}, EUNSUPPORTED),
    ({"total": 4}, {"dq_weight": 5 * _P + 2}, EINVAL),
    ({"total": 4, "positions": 0}, {}, EINVAL),
    ({"n_heads": 0}, {}, EINVAL),
])
def test_backward_checks(kw, grad, want):
    a, g = _args(**kw), _grad(**grad)
    assert _abi.lib().ifa4_qk_norm_rope_bwd(ctypes.byref(a), ctypes.byref(g), None, 0,
                                            None) == want


@pytest.mark.parametrize("kw", [dict(n_heads=(1 << 31) - 1), dict(kv_heads=(1 << 31) - 1),
                                dict(n_heads=(1 << 31) - 1, kv_heads=(1 << 31) - 1)])
def test_more_heads_than_the_launch_counts(kw):
    a, g = _args(total=1, **kw), _grad()
    lib = _abi.lib()
    assert lib.ifa4_qk_norm_rope_fwd(ctypes.byref(a), None) == EUNSUPPORTED
    assert lib.ifa4_qk_norm_rope_bwd_workspace_bytes(ctypes.byref(a)) == 0
    assert lib.ifa4_qk_norm_rope_bwd(ctypes.byref(a), ctypes.byref(g), None, 0, None) == EUNSUPPORTED


def test_backward_workspace():
    size = _abi.lib().ifa4_qk_norm_rope_bwd_workspace_bytes
    row = 2 * 128 * 4  # of a workgroup: 16 tokens at d 128, and two of the ten heads
    assert size(ctypes.byref(_args(total=1))) == 5 * row
    assert size(ctypes.byref(_args(total=33))) == 3 * 5 * row
    assert size(ctypes.byref(_args(total=16 * 300))) == 300 * 2 * row  # five heads
    assert size(ctypes.byref(_args(total=16 * 500))) == 500 * row      # all heads
    assert size(ctypes.byref(_args(total=1, q_weight=0, k_weight=0))) == 0
    assert size(ctypes.byref(_args(total=9, n_heads=0, kv_heads=0))) == 0
    assert size(ctypes.byref(_args(total=9, n_heads=0))) == 0
    most = size(ctypes.byref(_args(total=(1 << 31) - 1)))
    assert most == size(ctypes.byref(_args(total=1 << 24)))
    short = ctypes.c_void_p(_P)
    for ws, n in ((short, 5 * row - 1), (ctypes.c_void_p(_P + 64), 1 << 20)):
        assert _abi.lib().ifa4_qk_norm_rope_bwd(ctypes.byref(_args(total=1)), ctypes.byref(_grad()),
                                                ws, n, None) == EWORKSPACE


def _append(**kw):
    base = dict(kv_dtype=_abi.IFA4_BF16, v=_P, v_stride_t=256, v_stride_h=128, k_cache=2 * _P,
                v_cache=3 * _P, k_cache_stride_t=256, k_cache_stride_h=128, v_cache_stride_t=256,
                v_cache_stride_h=128, cu_seqlens=4 * _P, batch=2)
    return _abi.make_kv_append(**dict(base, **kw))


def _kv(**kw):
    base = dict(block_size=16, block_table=_P, seqused_k=2 * _P, block_table_stride=4,
                k_stride_block=4096, v_stride_block=4096, num_blocks=8, max_blocks_per_seq=4)
    return _abi.make_paged(**dict(base, **kw))


FP8 = {"kv_dtype": _abi.IFA4_FP8_E4M3}


@pytest.mark.parametrize("kw,append,kv,want", [(a, {}, {}, w) for a, w in SHARED] + [
    ({"n_heads": 0, "q": 0, "q_out": 0}, {}, {}, OK),
    ({"kv_heads": 0}, {}, {}, EINVAL),
    ({"total": 4, "q_out": 0}, {}, {}, EINVAL),
    ({}, {"struct_size": 8}, {}, EINVAL),
    ({}, {}, {"struct_size": 8}, EINVAL),
    ({}, {"batch": -1}, {}, EINVAL),
    ({}, {"kv_dtype": _abi.IFA4_FP16}, {}, EUNSUPPORTED),
    ({}, dict(FP8, k_scale=0.0), {}, EINVAL),
    ({}, dict(FP8, v_scale=float("inf")), {}, EINVAL),
    ({}, dict(FP8, v_scale=1e-40), {}, EINVAL),        # its reciprocal overflows
    ({}, {"k_scale": 0.0}, {}, OK),                    # not read for a 16-bit cache
    ({}, {}, {"block_size": 12}, EINVAL),
    ({}, {}, {"block_size": 4}, EINVAL),
    ({}, {}, {"num_blocks": -1}, EINVAL),
    ({"total": 4}, {"v": 0}, {}, EINVAL),
    ({"total": 4}, {"v": _P + 2}, {}, EUNSUPPORTED),
    ({"total": 4}, {"k_cache": 0}, {}, EINVAL),
    ({"total": 4}, {"cu_seqlens": 0}, {}, EINVAL),
    ({"total": 4}, {}, {"block_table": 0}, EINVAL),
    ({"total": 4}, {}, {"seqused_k": 2}, EINVAL),
    ({"total": 4}, {}, {"num_blocks": 0}, EINVAL),
    ({"total": 4}, {}, {"max_blocks_per_seq": 1 << 27}, EUNSUPPORTED),
    ({"total": 4}, {"k_cache_stride_t": 260}, {}, EUNSUPPORTED),
    ({"total": 4}, dict(FP8, k_cache_stride_t=264), {}, EUNSUPPORTED),  # 16 bytes: 16 elements
    ({"total": 4}, {"v_cache_stride_h": 64}, {}, EUNSUPPORTED),
    ({"total": 4}, {"v_cache": 3 * _P + 8}, {}, EUNSUPPORTED),
    ({"total": 4}, {"batch": 0}, {}, OK),              # tokens of no sequence: nothing to write
])
def test_append_checks(kw, append, kv, want):
    a, ap, pk = _args(**kw), _append(**append), _kv(**kv)
    assert _abi.lib().ifa4_kv_append_paged(ctypes.byref(a), ctypes.byref(ap), ctypes.byref(pk),
                                           None) == want


def test_python_refusals_without_a_gpu():
    q, k = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="nothing to do"):
        inkling_fa4_qk_norm_rope(q, k)
    cos = torch.ones(8, 32, requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        inkling_fa4_qk_norm_rope(q, k, cos=cos, sin=cos, positions=torch.zeros(3, dtype=torch.int32))
    w = torch.ones(64)
    with pytest.raises(NotImplementedError):  # CPU tensors: there is no CPU kernel
        inkling_fa4_qk_norm_rope(q, k, w, w)
    cache = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    ints = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        inkling_fa4_kv_append_paged(k, k, cache, cache.clone(), ints, ints[:1], ints[None])


ODD = dict(q_stride_t=67, k_stride_t=67, q_stride_h=3, k_stride_h=3)


@pytest.mark.parametrize("kw,want", [
    ({"total": 1, "n_heads": 1, "kv_heads": 1}, EWORKSPACE),  # every check passed
    ({"total": 2, "n_heads": 1, "kv_heads": 1}, EUNSUPPORTED),
    ({"total": 1, "n_heads": 2, "kv_heads": 1}, EUNSUPPORTED),
    ({"total": 1, "n_heads": 1, "kv_heads": 2}, EUNSUPPORTED),
])
def test_strides_of_dimensions_of_one(kw, want):
    """They are not looked at (the backward pass asks for its workspace last); others are."""
    a, g = _args(**kw, **ODD), _grad(gq_stride_t=5, gk_stride_t=5, dq_stride_t=9, dk_stride_t=9,
                                     gq_stride_h=128 + 3 * (kw["n_heads"] == 1))
    assert _abi.lib().ifa4_qk_norm_rope_bwd(ctypes.byref(a), ctypes.byref(g), None, 0, None) == want


@pytest.mark.parametrize("kw,append,kv", [
    ({"kv_heads": 2}, dict(k_cache_stride_h=132), {}),
    ({"kv_heads": 1}, {}, dict(num_blocks=2, k_stride_block=4100)),
    ({"kv_heads": 1}, dict(k_cache_stride_t=132), {}),
])
def test_cache_strides_that_are_stepped_along(kw, append, kv):
    a = _args(total=1, n_heads=1, **kw)
    ap, pk = _append(**append), _kv(**dict(dict(num_blocks=1), **kv))
    assert _abi.lib().ifa4_kv_append_paged(ctypes.byref(a), ctypes.byref(ap), ctypes.byref(pk),
                                           None) == EUNSUPPORTED
