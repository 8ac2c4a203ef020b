"""Prefill over a paged cache: ragged batches whose ranges are cut into chunks, and what lies past
the last key that a tile of queries sees."""
import ctypes
import math

import pytest
import torch

from inkling_fa4 import _abi, inkling_fa4_rel_attention_paged
from paged_cases import F8, Case

pytestmark = pytest.mark.gpu

# Sequences of one, two and three chunks of 50 key tiles (3200 keys) beside each other, lengths next
# to the chunks' edges, a sequence without keys, one without queries, one with more queries than keys.
NEWS = [500, 3, 120, 300, 77, 1, 256, 40, 0, 129, 5, 200, 64, 333, 20, 2]
LENS = [8000, 90, 3100, 6500, 3300, 7999, 256, 0, 4000, 6400, 3, 3200, 3201, 5000, 6401, 7000]


def run(c, dev, max_q=None, max_k=None):
    print("paged plans:", c.told(), flush=True)
    out, lse = inkling_fa4_rel_attention_paged(*c.on(dev), max_q or c.max_q, max_k or c.max_k,
                                               c.extent, causal=c.causal, **c.settings())
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu()


def chunks(c, max_q=None):
    """Chunks of the call's plan, by its workspace: partial rows of d values and an LSE in fp32."""
    p, total, d = 1 << 20, sum(c.news), c.d
    a = _abi.make_args(
        flags=_abi.IFA4_FLAG_BOTTOM_RIGHT, q=p, k=p, v=p, rel=p, out=p, cu_seqlens_q=p,
        q_stride_t=c.hq * d, q_stride_h=d, k_stride_t=c.hkv * d, k_stride_h=d, v_stride_t=c.hkv * d,
        v_stride_h=d, rel_stride_t=c.rel.stride(0), rel_stride_h=c.rel.stride(1),
        out_stride_t=c.hq * d, out_stride_h=d, total_q=total, batch=len(c.news), n_heads=c.hq,
        kv_heads=c.hkv, head_dim=d, rel_extent=c.extent, rel_width=c.rel.shape[2],
        max_seqlen_q=max_q or c.max_q, max_seqlen_k=c.max_k, softmax_scale=c.scale,
        window_left=c.window, causal=int(c.causal), qkv_dtype=_abi.IFA4_BF16, rel_dtype=_abi.IFA4_BF16)
    kv = _abi.make_paged(block_size=c.block, block_table=p, seqused_k=p,
                         block_table_stride=c.table.shape[1], k_stride_block=c.block * c.hkv * d,
                         v_stride_block=c.block * c.hkv * d, num_blocks=c.kc.shape[0],
                         max_blocks_per_seq=c.table.shape[1])
    quant = ctypes.byref(_abi.make_quant()) if c.kv == F8 else None
    n = _abi.lib().ifa4_prefill_paged_workspace_bytes(ctypes.byref(a), ctypes.byref(kv), quant)
    return round(n / (c.hq * total * (d + 1) * 4))


@pytest.mark.parametrize("kv", [None, F8])
@pytest.mark.parametrize("d,rel", [(128, "token"), (64, "table"), (64, "token"), (128, "table")])
def test_ragged_batch_in_chunks(cuda, kv, d, rel):
    c = Case(NEWS, LENS, d=d, rel=rel, kv=kv, seed=31)
    assert chunks(c) == 3
    got = run(c, cuda)
    c.check(got)
    again = run(c, cuda)
    assert all(torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.parametrize("kv", [None, F8])
def test_ragged_batch_in_chunks_not_causal(cuda, kv):
    c = Case(NEWS, LENS, dtype=torch.float16, rel_dtype=torch.float32, kv=kv, causal=False, extent=1024,
             seed=32)
    assert chunks(c) == 3
    c.check(run(c, cuda))


def test_equal_counts_under_a_loose_bound(cuda):
    """max_seqlen_q above every count: taken for a ragged batch, the same result."""
    c = Case([100] * 16, [6200] * 16, seed=33)
    assert chunks(c, 512) == 3
    c.check(run(c, cuda, max_q=512), seqs={0, 15})


@pytest.mark.parametrize("kv", [None, F8])
def test_ragged_batch_in_chunks_captured(cuda, kv):
    c, other = (Case(NEWS, LENS, kv=kv, seed=s) for s in (34, 35))
    args, new = c.on(cuda), other.on(cuda)

    def call():
        return inkling_fa4_rel_attention_paged(*args, c.max_q, c.max_k, c.extent, **c.settings())

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for rep in range(3):
        if rep == 1:
            for x, y in zip(args, new):
                if x.dtype == F8:
                    x, y = x.view(torch.uint8), y.view(torch.uint8)
                x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, call()))
        torch.cuda.synchronize()


# a tile of 128 rows ends inside a tile of 64 keys; packed heads; cut into chunks; a window
@pytest.mark.parametrize("news,lens,window", [([140], [150], -1), ([140, 300], [150, 333], -1),
                                              ([300], [5010], -1), ([300], [777], 100),
                                              ([200] * 5, [210] * 5, -1)])
@pytest.mark.parametrize("kv", [None, F8])
@pytest.mark.parametrize("rel", ["token", "table"])
def test_keys_that_no_query_of_a_tile_sees(cuda, news, lens, window, kv, rel):
    """Later tokens' keys and values may be infinite or NaN: the tiles before them do not notice."""
    c = Case(news, lens, window=window, kv=kv, rel=rel, seed=36)
    clean = run(c, cuda)
    for b, (n, lk) in enumerate(zip(news, lens)):
        past = lk - n + 128  # the first key past the first tile's last query
        j = torch.arange(past, lk)
        at = c.table[b, j // c.block].long()
        c.kc[at, j % c.block] = torch.tensor(math.nan).to(c.kc.dtype)
        c.vc[at, j % c.block] = torch.tensor(math.nan if kv else math.inf).to(c.vc.dtype)
    out, lse = run(c, cuda)
    start = 0
    for n in news:
        assert torch.equal(out[start:start + 128], clean[0][start:start + 128])
        assert torch.equal(lse[:, start:start + 128], clean[1][:, start:start + 128])
        start += n
