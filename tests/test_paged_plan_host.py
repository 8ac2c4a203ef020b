"""CPU tests of when a prefill over a paged cache is cut into chunks because its batch is ragged: the
workspace that the library asks for, on both sides of each condition."""
import ctypes

import pytest

from inkling_fa4 import _abi

P = 1 << 20
HQ, HKV, D = 8, 2, 128


def chunks(batch, total_q, max_q, max_k, window=-1, causal=1, fp8=False):
    """Chunks of the plan (0: not cut): partial rows of D values and one LSE in fp32."""
    a = _abi.make_args(
        flags=_abi.IFA4_FLAG_BOTTOM_RIGHT, q=P, k=P, v=P, rel=P, out=P, cu_seqlens_q=P,
        q_stride_t=HQ * D, q_stride_h=D, k_stride_t=HKV * D, k_stride_h=D, v_stride_t=HKV * D,
        v_stride_h=D, rel_stride_t=HQ * 128, rel_stride_h=128, out_stride_t=HQ * D, out_stride_h=D,
        total_q=total_q, batch=batch, n_heads=HQ, kv_heads=HKV, head_dim=D, rel_extent=128,
        rel_width=128, max_seqlen_q=max_q, max_seqlen_k=max_k, softmax_scale=0.1, window_left=window,
        causal=causal, qkv_dtype=_abi.IFA4_BF16, rel_dtype=_abi.IFA4_BF16)
    kv = _abi.make_paged(block_size=16, block_table=P, seqused_k=P, block_table_stride=4096,
                         k_stride_block=16 * HKV * D, v_stride_block=16 * HKV * D, num_blocks=2000,
                         max_blocks_per_seq=4096)
    quant = ctypes.byref(_abi.make_quant(k_scale=0.1, v_scale=0.1)) if fp8 else None
    n = _abi.lib().ifa4_prefill_paged_workspace_bytes(ctypes.byref(a), ctypes.byref(kv), quant)
    row = HQ * total_q * (D + 1) * 4
    assert n % 256 == 0 and 0 <= n - n // row * row < 512
    return n // row


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("causal", [0, 1])
def test_ragged_batches(fp8, causal):
    # 16 sequences of up to 500 queries: four tiles of 128 rows x 8 heads x 16 fill the 512 slots,
    # so that the plan for equal lengths leaves the call whole
    for total_q in (16, 2050, 4000, 7499):
        assert chunks(16, total_q, 500, 8000, causal=causal, fp8=fp8) == 3
    assert chunks(32, 8000, 500, 8000, causal=causal, fp8=fp8) == 3


def test_each_condition():
    assert chunks(16, 4000, 500, 8000) == 3
    # counts that fill 15/16 of the bound are equal ones
    assert chunks(16, 7500, 500, 8000) == 0 and chunks(16, 8000, 500, 8000) == 0
    # 96 tiles of 64 keys
    assert chunks(16, 4000, 500, 95 * 64) == 0 and chunks(16, 4000, 500, 95 * 64 + 1) == 3
    # a window keeps every range short
    assert chunks(16, 4000, 500, 8000, window=511) == 0
    # one and a half resident rounds of live workgroups (of 512): (total / 128 + batch / 2) heads
    assert chunks(48, 72 * 128 + 127, 500, 8000) == 3 and chunks(48, 73 * 128, 500, 8000) == 0
    # one sequence is not ragged
    assert chunks(1, 4000, 8192, 16384) == 0


@pytest.mark.parametrize("max_k", [6145, 6400, 8000, 20000, 65536])
def test_three_chunks_cover_the_longest_range(max_k):
    tiles = -(-max_k // 64)
    assert 3 * (2 * tiles // 5) >= tiles
    assert chunks(16, 4000, 500, max_k) == 3
