"""A key of NaN that a row sees makes both of the row's results NaN: an LSE of -inf beside it
would tell a caller that merges partial results that the row has no keys."""
import math

import pytest
import torch

from inkling_fa4 import inkling_fa4_rel_attention_sparse_paged
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


def check(c, rows, got, clean):
    print("nan rows:", c.told(), flush=True)
    (out, lse), (out0, lse0) = ([x.cpu() for x in r] for r in (got, clean))
    assert rows.any() and not rows.all()
    assert out[rows].isnan().all() and lse.t()[rows].isnan().all()
    assert torch.equal(out[~rows], out0[~rows]) and torch.equal(lse.t()[~rows], lse0.t()[~rows])


def both(c, hits, dev, call):
    clean = call(*c.on(dev))
    rows = spoil(c, hits)
    got = call(*c.on(dev))
    torch.cuda.synchronize()
    check(c, rows, got, clean)


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
