"""A key of NaN that a row sees makes both of the row's results NaN: an LSE of -inf beside it
would tell a caller that merges partial results that the row has no keys.  Every attention
operator, in the forms that a call can take (one pass, shares joined by a second)."""
import math

import pytest
import torch

from inkling_fa4 import (inkling_fa4_rel_attention, inkling_fa4_rel_attention_decode,
                         inkling_fa4_rel_attention_decode_paged,
                         inkling_fa4_rel_attention_decode_shared_prefix,
                         inkling_fa4_rel_attention_paged, inkling_fa4_rel_attention_rproj,
                         inkling_fa4_rel_attention_sparse_paged)
from paged_cases import F8, Case

pytestmark = pytest.mark.gpu


def put(c, seq, key, kvh, x):
    c.kc[int(c.table[seq, key // c.block]), key % c.block, kvh] = torch.tensor(x).to(c.kc.dtype)


def spoil(c, hits):
    """NaN in the keys (sequence, key, kv head); the rows [total_q, hq] that see one of them."""
    rows = torch.zeros(sum(c.news), c.hq, dtype=torch.bool)
    group = c.hq // c.hkv
    for seq, key, kvh in hits:
        put(c, seq, key, kvh, math.nan)
        start = sum(c.news[:seq])
        see = c.visible(seq)[0][:, key]
        rows[start:start + c.news[seq], kvh * group:(kvh + 1) * group] |= see[:, None]
    return rows


def tiles(c, hits):
    """Rows of the sequences and heads of the hits: those beside a row that sees a hit which they do
    not see are unspecified in the prefill, whose tiles of queries take finite keys only."""
    rows = torch.zeros(sum(c.news), c.hq, dtype=torch.bool)
    group = c.hq // c.hkv
    for seq, _, kvh in hits:
        start = sum(c.news[:seq])
        rows[start:start + c.news[seq], kvh * group:(kvh + 1) * group] = True
    return rows


def check(c, rows, got, clean, beside):
    print("nan rows:", c.told(), flush=True)
    (out, lse), (out0, lse0) = ([x.cpu() for x in r] for r in (got, clean))
    assert rows.any() and not rows.all()
    assert out[rows].isnan().all() and lse.t()[rows].isnan().all()
    same = ~(rows | beside)
    assert torch.equal(out[same], out0[same]) and torch.equal(lse.t()[same], lse0.t()[same])


def both(c, hits, dev, call, tiled=False):
    clean = call(*c.on(dev))
    rows = spoil(c, hits)
    got = call(*c.on(dev))
    torch.cuda.synchronize()
    check(c, rows, got, clean, tiles(c, hits) if tiled else torch.zeros_like(rows))


# sequences x tokens x list: one wave a list, some waves, lists shared by several workgroups
@pytest.mark.parametrize("news,lens,top", [([700, 600], [700, 900], 4), ([20, 30], [500, 300], 40),
                                           ([1, 1, 1], [1900, 700, 2000], 130)])
@pytest.mark.parametrize("kv", [None, F8])
def test_sparse(cuda, news, lens, top, kv):
    c = Case(news, lens, kv=kv, seed=top)
    lists = torch.arange(top, dtype=torch.int32, device=cuda).expand(sum(news), c.hkv, top).contiguous()

    def call(*a):
        return inkling_fa4_rel_attention_sparse_paged(*a, lists, c.max_q, c.max_k, c.extent,
                                                      **c.settings())

    both(c, [(0, 0, 1), (1, 16 * min(top, 15) + 3 if top > 4 else 40, 0)], cuda, call)


@pytest.mark.parametrize("lens", [[700, 90], [3000, 2500]])
def test_sparse_rows_of_nothing_but_nan(cuda, lens):
    """Every listed key is NaN: the maximum stays -inf, the row is NaN all the same."""
    c = Case([1, 1], lens, seed=3)
    lists = torch.arange(60, dtype=torch.int32, device=cuda).expand(2, c.hkv, 60).contiguous()

    def call(*a):
        return inkling_fa4_rel_attention_sparse_paged(*a, lists, c.max_q, c.max_k, c.extent,
                                                      **c.settings())

    both(c, [(0, j, 0) for j in range(lens[0])], cuda, call)


# one pass, packed heads, few tiles cut into chunks, a ragged batch cut into chunks
PREFILLS = [([100, 3], [100, 90]), ([4, 3], [1000, 700]), ([128, 40], [3000, 2000]),
            ([500] + [60] * 15, [7000] + [500] * 15)]


@pytest.mark.parametrize("news,lens", PREFILLS)
@pytest.mark.parametrize("kv", [None, F8])
def test_paged_prefill(cuda, news, lens, kv):
    c = Case(news, lens, kv=kv, seed=len(news))

    def call(*a):
        return inkling_fa4_rel_attention_paged(*a, c.max_q, c.max_k, c.extent, **c.settings())

    both(c, [(0, 0, 1), (1, 5, 0)], cuda, call, tiled=True)


def contiguous(c, kc, vc, table):
    """K and V of a case's sequences one after the other, and their offsets."""
    k, v = (torch.cat([x[table[b, torch.arange(lk, device=x.device) // c.block].long(),
                         torch.arange(lk, device=x.device) % c.block]
                       for b, lk in enumerate(c.lens)]) for x in (kc, vc))
    cu = torch.tensor([0] + c.lens, dtype=torch.int32).cumsum(0).to(torch.int32)
    return k, v, cu.to(k.device)


@pytest.mark.parametrize("news,lens", PREFILLS[:3] + [([500, 300], [9000, 200])])
def test_prefill(cuda, news, lens):
    c = Case(news, lens, seed=7)

    def call(q, kc, vc, rel, cu, used, table):
        k, v, cu_k = contiguous(c, kc, vc, table)
        return inkling_fa4_rel_attention(q, k, v, rel, cu, cu_k, c.max_q, c.max_k, c.extent,
                                         softmax_scale=c.scale, return_lse=True, bottom_right=True)

    both(c, [(0, 0, 1), (1, 5, 0)], cuda, call, tiled=True)


@pytest.mark.parametrize("news,lens", [([100, 3], [100, 90]), ([128, 40], [3000, 2000])])
def test_projected_prefill(cuda, news, lens):
    c = Case(news, lens, seed=8)
    g = torch.Generator().manual_seed(8)
    r = torch.randn(sum(news), c.hq, 16, generator=g).to(cuda)
    w = torch.randn(16, c.extent, generator=g).to(cuda)

    def call(q, kc, vc, rel, cu, used, table):
        k, v, cu_k = contiguous(c, kc, vc, table)
        return inkling_fa4_rel_attention_rproj(q, k, v, r, w, cu, cu_k, c.max_q, c.max_k, c.extent,
                                               softmax_scale=c.scale, return_lse=True,
                                               bottom_right=True)

    both(c, [(0, 0, 1), (1, 5, 0)], cuda, call, tiled=True)


# one launch, and waves whose partials are combined
@pytest.mark.parametrize("lens", [[300, 90], [9000, 5000, 70]])
@pytest.mark.parametrize("kv", [None, F8])
@pytest.mark.parametrize("paged", [False, True])
def test_decode(cuda, lens, kv, paged):
    c = Case([1] * len(lens), lens, kv=kv, seed=9)

    def call(q, kc, vc, rel, cu, used, table):
        if paged:
            return inkling_fa4_rel_attention_decode_paged(
                q, kc, vc, rel, cu, used, table, 1, c.max_k, c.extent, bottom_right=True, **c.settings())
        raw = [x.view(torch.uint8) if kv else x for x in (kc, vc)]
        k, v, cu_k = contiguous(c, *raw, table)
        return inkling_fa4_rel_attention_decode(q, k.view(kc.dtype), v.view(kc.dtype), rel, cu, cu_k, 1,
                                                c.max_k, c.extent, bottom_right=True, **c.settings())

    both(c, [(0, 0, 1), (1, 60, 0)], cuda, call)


@pytest.mark.parametrize("kv", [None, F8])
def test_shared_prefix_decode(cuda, kv):
    c = Case([1, 1, 1], [900, 700, 40], kv=kv, seed=10)

    def call(q, kc, vc, rel, cu, used, table):
        return inkling_fa4_rel_attention_decode_shared_prefix(
            q, kc, vc, rel, cu, used, table, table[0, :2].contiguous(), 0, 1, c.max_k, c.extent,
            **c.settings())

    both(c, [(0, 0, 1), (1, 60, 0)], cuda, call)
