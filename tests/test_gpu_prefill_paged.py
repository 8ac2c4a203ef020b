"""Prefill over a paged cache on the GPU against the definition in 64 bits (bounds in
paged_cases) and against the contiguous prefill."""
import math

import pytest
import torch

from inkling_fa4 import (inkling_fa4_kv_append_paged, inkling_fa4_rel_attention,
                         inkling_fa4_rel_attention_decode_paged, inkling_fa4_rel_attention_paged)
from paged_cases import F8, Case

pytestmark = pytest.mark.gpu


def run(c, dev, **kw):
    print("prefill paged:", c.told(), flush=True)
    out, lse = inkling_fa4_rel_attention_paged(*c.on(dev), c.max_q, c.max_k, c.extent,
                                               causal=c.causal, **dict(c.settings(), **kw))
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu()


NEWS = [1, 5, 64, 130, 33, 2, 200, 0, 17]
LENS = [1, 300, 64, 700, 1000, 17, 200, 90, 2049]


@pytest.mark.parametrize("block", [8, 16, 32, 64, 256])
@pytest.mark.parametrize("kv", [None, F8])
def test_blocks(cuda, block, kv):
    c = Case(NEWS, LENS, block=block, kv=kv, seed=block)
    c.check(run(c, cuda))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (8, 2, 128), (16, 1, 128), (6, 2, 64), (5, 5, 128),
                                      (32, 1, 64), (7, 1, 128)])
@pytest.mark.parametrize("kv", [None, F8])
def test_heads(cuda, hq, hkv, d, dtype, kv):
    c = Case([3, 100, 20], [500, 163, 900], hq, hkv, d, dtype, kv=kv, seed=hq + d)
    c.check(run(c, cuda))


@pytest.mark.parametrize("rel", ["token", "table"])
@pytest.mark.parametrize("rel_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("extent,width", [(1, 1), (17, 40), (128, 128), (1024, 1025)])
@pytest.mark.parametrize("kv", [None, F8])
def test_biases(cuda, rel, rel_dtype, extent, width, kv):
    c = Case([70, 1, 9], [700, 40, 1200], rel=rel, rel_dtype=rel_dtype, extent=extent, width=width,
             kv=kv, seed=extent)
    c.check(run(c, cuda))


def test_no_bias(cuda):
    c = Case([70, 1, 9], [700, 40, 1200], extent=0, width=0)
    c.check(run(c, cuda))


@pytest.mark.parametrize("window", [0, 1, 31, 63, 64, 200, 700, 5000, 2 ** 31 - 1])
@pytest.mark.parametrize("kv", [None, F8])
def test_windows(cuda, window, kv):
    c = Case(NEWS, LENS, window=window, kv=kv, seed=3)
    c.check(run(c, cuda))


@pytest.mark.parametrize("window", [-1, 40])
@pytest.mark.parametrize("kv", [None, F8])
def test_not_causal(cuda, window, kv):
    c = Case(NEWS, LENS, window=window, causal=False, kv=kv, seed=4)
    c.check(run(c, cuda))


@pytest.mark.parametrize("kv", [None, F8])
def test_more_queries_than_keys_and_empty_sequences(cuda, kv):
    """The first queries see nothing; a sequence without keys, one without queries."""
    c = Case([5, 140, 3, 0, 1, 4], [3, 64, 0, 0, 0, 300], kv=kv, seed=5)
    c.check(run(c, cuda))
    c = Case([4, 4], [0, 0], kv=kv)
    c.check(run(c, cuda))
    c = Case([0, 0], [20, 30], kv=kv)
    out, lse = run(c, cuda)
    assert out.shape == (0, 8, 128) and lse.shape == (8, 0)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("news,lens", [([4] * 8, [1000] * 8), ([512], [9000]), ([2] * 40, [3000] * 40),
                                       ([300, 7], [5000, 11000]), ([128] * 6, [128] * 6)])
def test_split_and_packed(cuda, news, lens, d):
    """Few tiles over long caches (cut into chunks, merged) and short queries (packed rows)."""
    for kv in (None, F8):
        c = Case(news, lens, d=d, kv=kv, extent=100, seed=len(news))
        c.check(run(c, cuda), seqs={0, len(news) - 1})


@pytest.mark.parametrize("layout", ["heads", "joint"])
@pytest.mark.parametrize("kv", [None, F8])
def test_cache_layouts(cuda, layout, kv):
    c = Case(NEWS, LENS, layout=layout, kv=kv, seed=6)
    c.check(run(c, cuda))


@pytest.mark.parametrize("kv", [None, F8])
@pytest.mark.parametrize("window", [10, 100])
def test_blocks_left_behind_by_the_window(cuda, window, kv):
    """Keys left of every query's window may be infinite or NaN, and their blocks gone."""
    c = Case([1, 30, 150], [400, 1000, 700], window=window, kv=kv, seed=7)
    for b, (n, lk) in enumerate(zip(c.news, c.lens)):
        first = max(0, lk - n - window)
        j = torch.arange(first)
        at = c.table[b, j // c.block].long()
        c.kc[at, j % c.block] = torch.tensor(math.nan).to(c.kc.dtype)
        c.vc[at, j % c.block] = torch.tensor(math.nan if kv else math.inf).to(c.vc.dtype)
    got = run(c, cuda)
    for x in (c.kc, c.vc):  # the definition multiplies unseen values by zero
        x.copy_(torch.nan_to_num(x.float(), 0.0, 0.0, 0.0).to(x.dtype))
    c.check(got)
    for b, (n, lk) in enumerate(zip(c.news, c.lens)):
        c.table[b, :max(0, lk - n - window) // c.block] = -7
    c.check(run(c, cuda))


def test_entries_outside_the_pool_read_as_zero(cuda):
    for kv in (None, F8):
        c = Case(NEWS, LENS, kv=kv, seed=8)
        c.table[3, 4], c.table[4, 0], c.table[6, 12], c.table[8, 100] = -1, 1 << 20, -(1 << 31), c.kc.shape[0]
        c.check(run(c, cuda))


def test_lengths_past_the_table_are_cut(cuda):
    c = Case([4, 4], [100, 64], seed=9)
    want = run(c, cuda)
    c.table = c.table[:, :7].contiguous()  # 112 keys
    c.used = torch.tensor([112, 64], dtype=torch.int32)
    whole = run(c, cuda)
    c.used = torch.tensor([1 << 30, 64], dtype=torch.int32)
    cut = run(c, cuda)
    assert torch.equal(whole[0][4:], want[0][4:])
    assert torch.equal(torch.nan_to_num(whole[0]), torch.nan_to_num(cut[0]))
    c.used = torch.tensor([-5, 64], dtype=torch.int32)
    none = run(c, cuda)
    assert not none[0][:4].any() and none[1][:, :4].isneginf().all()
    assert torch.equal(none[0][4:], want[0][4:])


@pytest.mark.parametrize("news,lens", [(NEWS, LENS), ([512], [2500]), ([3] * 70, list(range(60, 760, 10)))])
def test_as_the_contiguous_prefill(cuda, news, lens):
    c = Case(news, lens, seed=10, extent=200)
    q, kc, vc, rel, cu, used, table = c.on(cuda)
    got = run(c, cuda)
    k, v = (torch.cat([x[table[b, torch.arange(lk, device=cuda) // c.block].long(),
                         torch.arange(lk, device=cuda) % c.block] for b, lk in enumerate(lens)])
            for x in (kc, vc))
    cu_k = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32).to(cuda)
    want = inkling_fa4_rel_attention(q, k, v, rel, cu, cu_k, c.max_q, c.max_k, c.extent,
                                     softmax_scale=c.scale, return_lse=True, bottom_right=True)
    torch.testing.assert_close(got[0].float(), want[0].cpu().float(), atol=1e-3, rtol=1e-2)
    torch.testing.assert_close(got[1], want[1].cpu(), atol=1e-5, rtol=0)


def test_one_query_as_the_paged_decode(cuda):
    lens = [1, 16, 17, 500, 4000]
    for kv in (None, F8):
        c = Case([1] * 5, lens, kv=kv, seed=11)
        got = run(c, cuda)
        want = inkling_fa4_rel_attention_decode_paged(*c.on(cuda), 1, c.max_k, c.extent,
                                                      bottom_right=True, **c.settings())
        torch.testing.assert_close(got[0].float(), want[0].cpu().float(), atol=1e-3, rtol=1e-2)
        torch.testing.assert_close(got[1], want[1].cpu(), atol=2e-5, rtol=0)


def test_prompt_in_chunks(cuda):
    """Append and attend chunk by chunk: what one prefill of the whole prompt gives."""
    g = torch.Generator(cuda).manual_seed(12)
    n, hq, hkv, d, block, extent = 700, 8, 2, 128, 16, 256
    q, k, v = (torch.randn(n, h, d, generator=g, device=cuda).bfloat16() for h in (hq, hkv, hkv))
    rel = (0.5 * torch.randn(n, hq, extent, generator=g, device=cuda)).bfloat16()
    table = torch.randperm(60, generator=g, device=cuda).to(torch.int32)[:44].view(1, 44)
    kc, vc = (torch.full((60, block, hkv, d), math.nan, device=cuda).bfloat16() for _ in range(2))

    def i32(*x):
        return torch.tensor(x, dtype=torch.int32, device=cuda)

    outs, at = [], 0
    for m in (1, 100, 256, 7, 336):
        part = slice(at, at + m)
        at += m
        inkling_fa4_kv_append_paged(k[part], v[part], kc, vc, i32(0, m), i32(at), table)
        outs.append(inkling_fa4_rel_attention_paged(q[part], kc, vc, rel[part], i32(0, m), i32(at),
                                                    table, m, at, extent))
    want = inkling_fa4_rel_attention(q, k, v, rel, i32(0, n), i32(0, n), n, n, extent)
    torch.testing.assert_close(torch.cat(outs).float(), want.float(), atol=1e-3, rtol=1e-2)


def test_far_blocks(cuda):
    """A pool of more than 2^32 elements, blocks at both ends."""
    hkv, d, block = 2, 128, 16
    blocks = (1 << 32) // (block * hkv * d) + 64
    lens, news = [200, 90], [20, 90]
    for kv in (None, F8):
        c = Case(news, lens, kv=kv, seed=13)
        _, k, v, *_ = c.on(cuda)
        far = c.table.clone()
        high = torch.arange(c.table.shape[1]) % 2 == 0
        good = c.table < c.kc.shape[0]
        far[:, high] = torch.where(good, far + blocks - c.kc.shape[0], far)[:, high]
        big = []
        for x in (k, v):
            pool = torch.empty((blocks,) + x.shape[1:], dtype=x.dtype, device=cuda)
            raw, src = pool.view(torch.uint8), x.view(torch.uint8)
            raw[:x.shape[0]] = src
            raw[-x.shape[0]:] = src
            big.append(pool)
        args = c.on(cuda)
        args[1:3], args[6] = big, far.to(cuda)
        out, lse = inkling_fa4_rel_attention_paged(*args, c.max_q, c.max_k, c.extent, **c.settings())
        torch.cuda.synchronize()
        c.check((out.cpu(), lse.cpu()))
        del big, args, pool, raw


def test_strided_queries_and_tables(cuda):
    c = Case(NEWS, LENS, seed=14)
    q, kc, vc, rel, cu, used, table = c.on(cuda)
    wide = torch.full((q.shape[0], 12, 160), math.nan, device=cuda).bfloat16()
    wide[:, 2:10, 16:144] = q
    rows = torch.full((table.shape[0], table.shape[1] + 9), -1, dtype=torch.int32, device=cuda)
    rows[:, 4:4 + table.shape[1]] = table
    wrel = torch.zeros(q.shape[0], 10, 150, device=cuda).bfloat16()
    wrel[:, 1:9, 7:135] = rel
    out, lse = inkling_fa4_rel_attention_paged(
        wide[:, 2:10, 16:144], kc, vc, wrel[:, 1:9, 7:135], cu, used, rows[:, 4:4 + table.shape[1]],
        c.max_q, c.max_k, c.extent, **c.settings())
    torch.cuda.synchronize()
    c.check((out.cpu(), lse.cpu()))


@pytest.mark.parametrize("kv", [None, F8])
@pytest.mark.parametrize("news,lens", [([3, 40], [900, 500]), ([4] * 3, [5000] * 3)])
def test_graph(cuda, kv, news, lens):
    """Captured once, replayed with other inputs; two captured calls share no workspace."""
    c, other = (Case(news, lens, kv=kv, seed=s) for s in (15, 16))
    args, new = c.on(cuda), other.on(cuda)

    def call(a):
        return inkling_fa4_rel_attention_paged(*a, c.max_q, c.max_k, c.extent, **c.settings())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = call(args)
        second = call([args[0] * 0.5] + args[1:])
    for rep in range(3):
        if rep == 1:
            for x, y in zip(args, new):
                if x.dtype == F8:
                    x, y = x.view(torch.uint8), y.view(torch.uint8)
                x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(first + second, call(args) + call([args[0] * 0.5] + args[1:])):
            assert torch.equal(got, want)
        torch.cuda.synchronize()


def test_stream(cuda):
    c = Case(NEWS, LENS, seed=17)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        args = c.on(cuda)
        out, lse = inkling_fa4_rel_attention_paged(*args, c.max_q, c.max_k, c.extent, **c.settings())
        out, lse = out.cpu(), lse.cpu()
    c.check((out, lse))


def test_rows_of_no_sequence(cuda):
    """Tokens past the last sequence stay as the allocation left them."""
    c = Case([5, 9], [50, 60], seed=18)
    args = c.on(cuda)
    args[0] = torch.cat([args[0], args[0][:3]])
    args[3] = torch.cat([args[3], args[3][:3]])
    torch.use_deterministic_algorithms(True)
    try:
        out, lse = inkling_fa4_rel_attention_paged(*args, c.max_q, c.max_k, c.extent, **c.settings())
    finally:
        torch.use_deterministic_algorithms(False)
    torch.cuda.synchronize()
    assert out[14:].isnan().all() and lse[:, 14:].isnan().all()
    c.check((out[:14].cpu(), lse[:, :14].cpu()))


def test_refusals(cuda):
    c = Case([3, 4], [40, 50], seed=19)
    args = c.on(cuda)

    def call(i=None, x=None, extent=c.extent, max_k=c.max_k, **kw):
        a = list(args)
        if i is not None:
            a[i] = x
        return inkling_fa4_rel_attention_paged(*a, c.max_q, max_k, extent, **dict(c.settings(), **kw))

    q, kc, vc, rel, cu, used, table = args
    for i, bad in [(0, q.float()), (0, q[:, :7]), (0, q.cpu()), (1, kc[0]), (1, kc.half()),
                   (1, kc[:, :12]), (2, vc[:-1]), (3, rel[:-1]), (3, rel.double()), (4, cu.long()),
                   (5, used[:1]), (5, used.long()), (6, table.long()), (6, table[:1]),
                   (6, table[:, ::2]), (1, kc[..., :100]), (2, vc.to(F8))]:
        with pytest.raises((ValueError, RuntimeError, IndexError)):
            call(i, bad)
    for kw in (dict(extent=c.extent + 1), dict(extent=-1), dict(softmax_scale=math.nan),
               dict(softmax_scale=0.0), dict(max_k=16 * table.shape[1] + 1)):
        with pytest.raises((ValueError, RuntimeError)):
            call(**kw)
    small = Case([3, 4], [40, 50], kv=F8, d=64, block=8)
    with pytest.raises(RuntimeError, match="EUNSUPPORTED"):  # a load of 16 rows needs one block
        inkling_fa4_rel_attention_paged(*small.on(cuda), small.max_q, small.max_k, small.extent,
                                        **small.settings())
    small = Case([3, 4], [40, 50], kv=F8)
    for kw in (dict(k_scale=0.0), dict(v_scale=-1.0), dict(k_scale=math.inf)):
        with pytest.raises(RuntimeError):
            inkling_fa4_rel_attention_paged(*small.on(cuda), small.max_q, small.max_k, small.extent,
                                            **dict(small.settings(), **kw))
    torch.cuda.synchronize()
