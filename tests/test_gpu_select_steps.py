"""The block choice for sequences of one to three new tokens, and over rows of more competing blocks
than a workgroup holds at once; against the definition in 64 bits."""
import math

import pytest
import torch

from inkling_fa4 import inkling_fa4_select_blocks_paged
from paged_cases import F8, Case
from test_gpu_sparse import key_like_bounds, run_select, want_lists

pytestmark = pytest.mark.gpu

STEPS = [([1, 1], [1500, 3000]), ([2, 1, 3], [700, 1500, 3000]), ([3, 0, 1], [2000, 500, 900])]


def check(c, b, dev, top=20, sink=1, recent=2, **kw):
    assert torch.equal(run_select(c, b, top, sink, recent, dev, **kw),
                       want_lists(c, b, top, sink, recent))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (8, 2, 128), (16, 1, 128), (6, 2, 64), (3, 1, 64),
                                      (40, 2, 128), (15, 3, 128), (5, 5, 128)])
@pytest.mark.parametrize("kv", [None, F8])
def test_heads(cuda, hq, hkv, d, dtype, kv):
    for i, (news, lens) in enumerate(STEPS):
        c = Case(news, lens, hq, hkv, d, dtype, kv=kv, seed=hq + d + i)
        check(c, key_like_bounds(c), cuda)


@pytest.mark.parametrize("block", [8, 16, 64])
@pytest.mark.parametrize("kv", [None, F8])
@pytest.mark.parametrize("top,sink,recent", [(1, 0, 1), (2, 1, 1), (9, 1, 2), (24, 0, 3), (40, 5, 5)])
def test_lists(cuda, block, kv, top, sink, recent):
    c = Case([2, 1, 3, 1], [700, 1500, 3000, 5], block=block, kv=kv, seed=top)
    check(c, key_like_bounds(c), cuda, top, sink, recent)


@pytest.mark.parametrize("kind", ["equal", "few", "zero", "signed zeros"])
@pytest.mark.parametrize("d,kv", [(128, None), (64, F8)])
def test_ties(cuda, kind, d, kv):
    for news, lens in STEPS:
        c = Case(news, lens, d=d, kv=kv, seed=9)
        b = key_like_bounds(c).float()
        if kind == "equal":
            b[:] = b[0].clone()
        elif kind == "few":
            b = b[torch.arange(b.shape[0]) % 5]
        else:
            b.zero_()
            if kind == "signed zeros":
                b[::2] = -0.0
        check(c, b.to(c.kc.dtype), cuda)


@pytest.mark.parametrize("d", [64, 128])
def test_near_ties(cuda, d):
    """Scores that differ past the 24th bit: large terms that cancel, small ones that decide.  The
    sums stay below 2^20, so 64 bits round them by 2^-33 at most; unequal scores differ by 2^-24 and
    more (q >= 1 times a step of the bound)."""
    for news, lens in STEPS:
        c = Case(news, lens, d=d, dtype=torch.float16, seed=10)
        c.q[:] = c.q.abs() + 1  # only upper bounds count
        g = torch.Generator().manual_seed(10)
        b = torch.zeros(c.kc.shape[0], c.hkv, 2, c.d).half()
        b[..., 1, 0], b[..., 1, 1] = 30000.0, -30000.0
        c.q[..., 0] = c.q[..., 1]
        b[..., 1, 2] = torch.randint(1, 2000, b.shape[:2], generator=g).half() * 2.0 ** -24
        check(c, b, cuda, 30)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("d,kv", [(64, None), (128, None), (128, F8)])
def test_infinite_and_nan(cuda, bad, d, kv):
    if kv and not math.isnan(bad):
        bad = math.copysign(448.0, bad)
    for news, lens in STEPS:
        c = Case(news, lens, d=d, kv=kv, seed=11)
        b = key_like_bounds(c).float()
        b[torch.rand(b.shape, generator=torch.Generator().manual_seed(11)) < 0.0005] = bad
        b = b.to(c.kc.dtype)
        check(c, b, cuda)
        c.q[1, 3, 7] = math.nan
        c.q[0, 6, 0] = math.inf
        check(c, b, cuda)


@pytest.mark.parametrize("kv", [None, F8])
def test_entries_outside_the_pool_and_loose_bounds(cuda, kv):
    c = Case([2, 1, 3], [700, 1500, 3000], kv=kv, seed=13)
    c.table[0, 5], c.table[1, 60], c.table[2, 100] = -1, 1 << 20, -(1 << 31)
    c.table[2, 101], c.table[2, 102] = c.kc.shape[0], (1 << 31) - 1
    b = key_like_bounds(c)
    check(c, b, cuda)
    check(c, b, cuda, max_k=c.table.shape[1] * c.block)
    # a bound of more tokens takes the way of longer chunks: the same lists
    check(c, b, cuda, max_q=200)


def test_strides(cuda):
    c = Case([2, 1, 3], [700, 1500, 3000], seed=14)
    b = key_like_bounds(c)
    q, _, _, _, cu, used, table = c.on(cuda)
    wide = torch.full((q.shape[0], 12, 160), math.nan, device=cuda).bfloat16()
    wide[:, 2:10, 16:144] = q
    pool = torch.full((b.shape[0], 5, 2, 128), math.nan, device=cuda).bfloat16()
    pool[:, 1:4:2] = b.to(cuda)
    rows = torch.full((3, table.shape[1] + 9), -1, dtype=torch.int32, device=cuda)
    rows[:, 4:-5] = table
    got = inkling_fa4_select_blocks_paged(wide[:, 2:10, 16:144], pool[:, 1:4:2], cu, used,
                                          rows[:, 4:-5], 16, c.max_q, c.max_k, 20)
    assert torch.equal(got.cpu(), want_lists(c, b, 20, 1, 2))


@pytest.mark.parametrize("news", [[1, 2], [4, 20]])
@pytest.mark.parametrize("kind", ["spread", "few", "equal", "step"])
def test_rows_of_more_than_a_round(cuda, news, kind):
    """More than 2048 competing blocks: equal scores on both sides of a round's border."""
    c = Case(news, [20000, 36000], block=8, hq=4, hkv=2, d=64, seed=15)
    b = key_like_bounds(c).float()
    if kind == "few":
        b = b[torch.arange(b.shape[0]) % 3]
    elif kind != "spread":
        b[:] = b[0].clone()
        if kind == "step":  # the best blocks sit across the border, the rest are equal
            for seq in range(2):
                b[c.table[seq, 2040:2060].long()] *= 1.5
    b = b.to(c.kc.dtype)
    for top in (30, 700, 2300):
        check(c, b, cuda, top)
