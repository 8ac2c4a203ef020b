"""Key bounds, block choice and attention over listed blocks on the GPU.  Bounds and choices are
compared for equality with their definitions (choices in 64 bits), the attention within the bounds
of paged_cases."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwad

from inkling_fa4 import (inkling_fa4_key_bounds_paged, inkling_fa4_kv_append_paged,
                         inkling_fa4_rel_attention_paged, inkling_fa4_rel_attention_sparse_paged,
                         inkling_fa4_select_blocks_paged)
from paged_cases import F8, Case

pytestmark = pytest.mark.gpu

NEWS = [1, 5, 64, 130, 33, 2, 200, 0, 17]
LENS = [1, 300, 64, 700, 1000, 17, 200, 90, 2049]


def same(a, b):
    """Equal, NaN to NaN."""
    a, b = a.float(), b.float()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


# ---- bounds -------------------------------------------------------------------------------------


def want_bounds(c, bounds):
    bounds = bounds.clone()
    for b, (n, lk) in enumerate(zip(c.news, c.lens)):
        n = min(n, lk)
        for blk in range((lk - n) // c.block, -(-lk // c.block)) if n else ():
            ent = int(c.table[b, blk])
            if 0 <= ent < c.kc.shape[0]:
                rows = c.kc[ent, :min(c.block, lk - blk * c.block)].float()
                bounds[ent, :, 0] = rows.amin(0).to(bounds.dtype)
                bounds[ent, :, 1] = rows.amax(0).to(bounds.dtype)
    return bounds


def run_bounds(c, bounds, dev, max_q=None):
    print("bounds:", c.told(), flush=True)
    _, kc, _, _, cu, used, table = c.on(dev)
    got = bounds.to(dev)
    inkling_fa4_key_bounds_paged(kc, got, cu, used, table, c.max_q if max_q is None else max_q)
    torch.cuda.synchronize()
    return got.cpu()


def some_bounds(c, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(c.kc.shape[0], c.hkv, 2, c.d, generator=g).to(c.kc.dtype)


@pytest.mark.parametrize("block", [8, 16, 32, 64, 256])
@pytest.mark.parametrize("kv", [None, F8])
@pytest.mark.parametrize("d,dtype", [(128, torch.bfloat16), (64, torch.float16)])
def test_bounds(cuda, block, kv, d, dtype):
    c = Case(NEWS, LENS, d=d, dtype=dtype, block=block, kv=kv, seed=block)
    old = some_bounds(c)
    assert same(run_bounds(c, old, cuda), want_bounds(c, old))


@pytest.mark.parametrize("hq,hkv", [(4, 4), (8, 1), (5, 5), (6, 3)])
@pytest.mark.parametrize("layout", ["heads", "joint"])
@pytest.mark.parametrize("kv", [None, F8])
def test_bounds_heads_and_layouts(cuda, hq, hkv, layout, kv):
    c = Case(NEWS, LENS, hq, hkv, layout=layout, kv=kv, seed=hq)
    old = some_bounds(c)
    assert same(run_bounds(c, old, cuda), want_bounds(c, old))


@pytest.mark.parametrize("block", [16, 128])
@pytest.mark.parametrize("kv", [None, F8])
def test_bounds_of_nan_and_infinite_keys(cuda, block, kv):
    c = Case([300, 40], [300, 500], block=block, kv=kv, seed=2)
    raw = c.kc.float()
    for i, x in enumerate((math.nan, 448.0 if kv else math.inf, -448.0 if kv else -math.inf)):
        raw[int(c.table[0, i % 2]), 3 + i, 1, 5 + i] = x
        raw[int(c.table[1, 499 // block]), 1, 0, 9 + i] = x
    c.kc = raw.to(c.kc.dtype)
    old = some_bounds(c)
    want = want_bounds(c, old)
    assert want.float().isnan().any()
    assert same(run_bounds(c, old, cuda), want)


def test_bounds_edges(cuda):
    """More new tokens than keys, none, entries outside the pool, lengths past the table."""
    c = Case([5, 140, 3, 0, 1, 4], [3, 64, 0, 0, 0, 300], seed=3)
    old = some_bounds(c)
    assert same(run_bounds(c, old, cuda), want_bounds(c, old))
    c = Case(NEWS, LENS, seed=4)
    c.table[3, 40], c.table[4, 62], c.table[6, 12] = -1, 1 << 20, c.kc.shape[0]
    assert same(run_bounds(c, some_bounds(c), cuda), want_bounds(c, some_bounds(c)))
    c = Case([4, 4], [100, 64], seed=5)
    c.table[0, 6] = -1
    c.used = torch.tensor([1 << 30, -7], dtype=torch.int32)
    old = some_bounds(c)
    assert same(run_bounds(c, old, cuda), old)  # the new tokens lie past the table, or nowhere


def test_bounds_refusals(cuda):
    c = Case([3, 4], [40, 50], seed=6)
    _, kc, _, _, cu, used, table = c.on(cuda)
    b = some_bounds(c).to(cuda)

    def call(k=kc, x=b, cu=cu, used=used, table=table, n=c.max_q):
        inkling_fa4_key_bounds_paged(k, x, cu, used, table, n)

    call()
    for kw in (dict(k=kc[0]), dict(k=kc.float()), dict(x=b.half()), dict(x=b[:-1]), dict(x=b[:, :1]),
               dict(x=b[..., :64]), dict(x=b.transpose(1, 2)), dict(k=kc.cpu()), dict(x=b.cpu()),
               dict(cu=cu.long()), dict(used=used[:1]), dict(table=table[:1]), dict(n=-1),
               dict(table=table[:, ::2]), dict(k=kc[:, :12], x=b), dict(x=b[:1].expand(b.shape))):
        with pytest.raises((RuntimeError, IndexError, ValueError)):
            call(**kw)
    with pytest.raises(RuntimeError, match="gradient"):
        call(x=b.clone().requires_grad_())
    with fwad.dual_level(), pytest.raises(NotImplementedError):
        call(k=fwad.make_dual(kc, torch.ones_like(kc)))
    before = b._version
    call()
    assert b._version > before  # autograd sees the change
    torch.cuda.synchronize()


# ---- choice -------------------------------------------------------------------------------------


def want_lists(c, bounds, top, sink, recent, total=None):
    """The choice by its definition, in 64 bits."""
    out = torch.full((sum(c.news) if total is None else total, c.hkv, top), -1, dtype=torch.int32)
    group, start = c.hq // c.hkv, 0
    for b, (n, lk) in enumerate(zip(c.news, c.lens)):
        nb = -(-lk // c.block)
        ent = c.table[b, :nb].long()
        good = (ent >= 0) & (ent < bounds.shape[0])
        bd = torch.where(good[:, None, None, None], bounds[torch.where(good, ent, 0)].double(), 0.0)
        for i in range(n):
            pos = lk - n + i
            cand = pos // c.block + 1 if pos >= 0 else 0
            for h in range(c.hkv):
                if cand <= top:
                    picked = list(range(cand))
                else:
                    q = c.q[start + i, h * group:(h + 1) * group].double()
                    mid = range(sink, cand - recent)
                    lo, hi = bd[sink:cand - recent, h, 0], bd[sink:cand - recent, h, 1]
                    score = (torch.where(q > 0, 0.0, q).sum(0) * lo
                             + torch.where(q < 0, 0.0, q).sum(0) * hi).sum(-1)
                    score = torch.where(score.isnan(), math.inf, score).tolist()
                    best = sorted(mid, key=lambda j: (-score[j - sink], j))[:top - sink - recent]
                    picked = list(range(sink)) + sorted(best) + list(range(cand - recent, cand))
                out[start + i, h, :len(picked)] = torch.tensor(picked, dtype=torch.int32)
        start += n
    return out


def run_select(c, bounds, top, sink, recent, dev, **kw):
    print("select:", c.told(), "top", top, sink, recent, flush=True)
    q, _, _, _, cu, used, table = c.on(dev)
    got = inkling_fa4_select_blocks_paged(
        q, bounds.to(dev), cu, used, table, c.block, kw.get("max_q", c.max_q),
        kw.get("max_k", c.max_k), top, sink_blocks=sink, recent_blocks=recent)
    torch.cuda.synchronize()
    return got.cpu()


def key_like_bounds(c, seed=0):
    return torch.sort(some_bounds(c, seed).float(), 2).values.to(c.kc.dtype)


@pytest.mark.parametrize("block", [8, 16, 64])
@pytest.mark.parametrize("kv", [None, F8])
@pytest.mark.parametrize("top,sink,recent", [(1, 0, 1), (2, 1, 1), (9, 1, 2), (24, 0, 3), (40, 5, 5),
                                             (300, 1, 2)])
def test_select(cuda, block, kv, top, sink, recent):
    c = Case(NEWS, LENS, block=block, kv=kv, seed=top)
    b = key_like_bounds(c)
    assert torch.equal(run_select(c, b, top, sink, recent, cuda), want_lists(c, b, top, sink, recent))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (8, 2, 128), (16, 1, 128), (6, 2, 64), (32, 1, 64),
                                      (40, 2, 128)])
@pytest.mark.parametrize("kv", [None, F8])
def test_select_heads(cuda, hq, hkv, d, dtype, kv):
    c = Case([3, 40, 1], [500, 640, 900], hq, hkv, d, dtype, kv=kv, seed=hq + d)
    b = key_like_bounds(c)
    assert torch.equal(run_select(c, b, 12, 1, 2, cuda), want_lists(c, b, 12, 1, 2))


@pytest.mark.parametrize("lens", [[6000] * 3, [70, 9000, 1, 0, 333], [40000]])
def test_select_steps(cuda, lens):
    """One token a sequence over long caches."""
    c = Case([1] * len(lens), lens, seed=len(lens))
    b = key_like_bounds(c)
    for top in (5, 64, 130):
        assert torch.equal(run_select(c, b, top, 1, 2, cuda), want_lists(c, b, top, 1, 2))


def test_select_many_sequences(cuda):
    lens = [50 + 37 * i % 900 for i in range(150)]
    c = Case([1] * 150, lens, seed=8)
    b = key_like_bounds(c)
    assert torch.equal(run_select(c, b, 8, 1, 2, cuda), want_lists(c, b, 8, 1, 2))


@pytest.mark.parametrize("kind", ["equal", "few", "zero", "signed zeros"])
def test_select_ties(cuda, kind):
    """Equal scores: the lower block."""
    c = Case([2, 20], [1500, 3000], seed=9)
    b = key_like_bounds(c)
    if kind == "equal":
        b[:] = b[0]
    elif kind == "few":
        b[:] = b[torch.arange(b.shape[0]) % 5]
    else:
        b.zero_()
        if kind == "signed zeros":
            b[::2] = -0.0
    assert torch.equal(run_select(c, b, 20, 1, 2, cuda), want_lists(c, b, 20, 1, 2))


def test_select_near_ties(cuda):
    """Scores that differ past the 24th bit: large terms that cancel, small ones that decide."""
    c = Case([1, 4], [3000, 3000], dtype=torch.float16, seed=10)
    c.q[:] = c.q.abs() + 1  # only upper bounds count
    g = torch.Generator().manual_seed(10)
    b = torch.zeros(c.kc.shape[0], c.hkv, 2, c.d).half()
    b[..., 1, 0], b[..., 1, 1] = 30000.0, -30000.0
    c.q[..., 0] = c.q[..., 1]
    b[..., 1, 2] = torch.randint(1, 2000, b.shape[:2], generator=g).half() * 2.0 ** -24
    assert torch.equal(run_select(c, b, 30, 1, 2, cuda), want_lists(c, b, 30, 1, 2))


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_select_infinite_and_nan_bounds(cuda, bad):
    c = Case([2, 20], [1500, 3000], seed=11)
    b = key_like_bounds(c)
    g = torch.Generator().manual_seed(11)
    hit = torch.rand(b.shape, generator=g) < 0.0005
    b[hit] = bad
    assert torch.equal(run_select(c, b, 20, 1, 2, cuda), want_lists(c, b, 20, 1, 2))
    c.q[1, 3, 7] = math.nan
    c.q[5, 6, 0] = math.inf
    assert torch.equal(run_select(c, b, 20, 1, 2, cuda), want_lists(c, b, 20, 1, 2))


def test_select_edges(cuda):
    """Tokens before the first key, of no sequence, entries outside the pool, loose lengths."""
    c = Case([5, 140, 3, 0, 1, 4], [3, 64, 0, 0, 0, 900], seed=12)
    b = key_like_bounds(c)
    want = want_lists(c, b, 3, 0, 1)
    assert torch.equal(run_select(c, b, 3, 0, 1, cuda), want)
    assert torch.equal(run_select(c, b, 3, 0, 1, cuda, max_q=200, max_k=912), want)
    c.q = torch.cat([c.q, c.q[:3]])
    got = run_select(c, b, 3, 0, 1, cuda)
    assert torch.equal(got[:-3], want) and (got[-3:] == -1).all()
    c = Case([2, 20], [1500, 3000], seed=13)
    c.table[0, 5], c.table[1, 100], c.table[1, 101] = -1, 1 << 20, c.kc.shape[0]
    b = key_like_bounds(c)
    assert torch.equal(run_select(c, b, 20, 1, 2, cuda), want_lists(c, b, 20, 1, 2))
    c = Case([0, 0], [20, 30])
    assert run_select(c, key_like_bounds(c), 3, 0, 1, cuda).shape == (0, 2, 3)


def test_select_without_sequences_or_queries(cuda):
    """Tokens of no sequence: -1 throughout, also where there is no sequence, or none has a query."""
    c = Case([2, 20], [1500, 3000], seed=13)
    q, _, _, _, cu, used, table = c.on(cuda)
    b = key_like_bounds(c).to(cuda)
    for cu2, n in ((cu[:1], 0), (torch.zeros_like(cu), 2)):
        got = inkling_fa4_select_blocks_paged(q, b, cu2, used[:n], table[:n], 16, 0, 3000, 20)
        assert got.shape == (22, 2, 20) and (got == -1).all()
    torch.cuda.synchronize()


def test_select_strides(cuda):
    c = Case([2, 20], [1500, 3000], seed=14)
    b = key_like_bounds(c)
    q, _, _, _, cu, used, table = c.on(cuda)
    wide = torch.full((q.shape[0], 12, 160), math.nan, device=cuda).bfloat16()
    wide[:, 2:10, 16:144] = q
    pool = torch.full((b.shape[0], 5, 2, 128), math.nan, device=cuda).bfloat16()
    pool[:, 1:4:2] = b.to(cuda)
    rows = torch.full((2, table.shape[1] + 9), -1, dtype=torch.int32, device=cuda)
    rows[:, 4:-5] = table
    got = inkling_fa4_select_blocks_paged(wide[:, 2:10, 16:144], pool[:, 1:4:2], cu, used,
                                          rows[:, 4:-5], 16, c.max_q, c.max_k, 20)
    assert torch.equal(got.cpu(), want_lists(c, b, 20, 1, 2))


def test_select_refusals(cuda):
    c = Case([3, 4], [400, 500], seed=15)
    q, _, _, _, cu, used, table = c.on(cuda)
    b = key_like_bounds(c).to(cuda)

    def call(q=q, b=b, cu=cu, used=used, table=table, block=16, max_q=c.max_q, max_k=c.max_k, top=5, **kw):
        inkling_fa4_select_blocks_paged(q, b, cu, used, table, block, max_q, max_k, top, **kw)

    call()
    for kw in (dict(q=q.float()), dict(q=q[:, :7]), dict(q=q.cpu()), dict(q=q[..., :64]), dict(b=b.half()),
               dict(b=b[:, :, :1]), dict(b=b.transpose(1, 2)), dict(b=b.cpu()), dict(cu=cu.long()),
               dict(used=used[:1]), dict(table=table[:1]), dict(table=table[:, ::2]), dict(block=12),
               dict(block=4), dict(block=0), dict(max_q=-1), dict(max_k=-1), dict(top=0), dict(top=2),
               dict(max_k=table.shape[1] * 16 + 1), dict(sink_blocks=-1), dict(recent_blocks=0),
               dict(sink_blocks=4), dict(b=b[:0])):
        with pytest.raises((RuntimeError, IndexError, ValueError)):
            call(**kw)
    torch.cuda.synchronize()


# ---- attention ----------------------------------------------------------------------------------


class Sparse(Case):
    """Lists drawn at random: sorted blocks up to the token's own, -1 behind them; messy=True mixes
    in entries to be passed over and blocks named twice, in any order."""

    def __init__(self, news, lens, top=8, messy=False, **kw):
        super().__init__(news, lens, **kw)
        g = torch.Generator().manual_seed(kw.get("seed", 0) + 1000)
        self.lists = torch.full((sum(news), self.hkv, top), -1, dtype=torch.int32)
        t = 0
        for b, (n, lk) in enumerate(zip(news, lens)):
            for i in range(n):
                own = max(0, (lk - n + i) // self.block + 1) if lk - n + i >= 0 else 0
                for h in range(self.hkv):
                    if messy:
                        pick = torch.randint(-3, own + 3, (top,), generator=g)
                        pick[pick == -2] = 1 << 30
                        pick[pick == -3] = -(1 << 31)
                    else:
                        pick = torch.randperm(own, generator=g)[:top].sort().values
                        if own and len(pick):
                            pick[-1] = own - 1
                    self.lists[t, h, :len(pick)] = pick.to(torch.int32)
                t += 1

    def times(self, b, h):
        start = sum(self.news[:b])
        n, lk = self.news[b], self.lens[b]
        nb = -(-lk // self.block)
        ls = self.lists[start:start + n, h].long()
        count = torch.zeros(n, nb + 1)
        ent = self.table[b, :nb].long()
        gone = (ent < 0) | (ent >= self.kc.shape[0])
        count.scatter_add_(1, torch.where((ls >= 0) & (ls < nb), ls, nb), torch.ones(ls.shape))
        count[:, :nb][:, gone] = 0
        return count[:, :nb].repeat_interleave(self.block, 1)[:, :lk]


def run(c, dev, lists=None, **kw):
    print("sparse:", c.told(), "lists", tuple(c.lists.shape), flush=True)
    out, lse = inkling_fa4_rel_attention_sparse_paged(
        *c.on(dev), (c.lists if lists is None else lists).to(dev), c.max_q, c.max_k, c.extent,
        **dict(c.settings(), **kw))
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu()


@pytest.mark.parametrize("block", [8, 16, 32, 64, 256])
@pytest.mark.parametrize("kv", [None, F8])
@pytest.mark.parametrize("messy", [False, True])
def test_sparse_blocks(cuda, block, kv, messy):
    c = Sparse(NEWS, LENS, top=7, messy=messy, block=block, kv=kv, seed=block)
    c.check(run(c, cuda))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (8, 2, 128), (16, 1, 128), (6, 2, 64), (5, 5, 128),
                                      (16, 1, 64), (7, 1, 128)])
@pytest.mark.parametrize("kv", [None, F8])
def test_sparse_heads(cuda, hq, hkv, d, dtype, kv):
    c = Sparse([3, 100, 20], [500, 163, 900], 6, hq=hq, hkv=hkv, d=d, dtype=dtype, kv=kv, seed=hq + d)
    c.check(run(c, cuda))


@pytest.mark.parametrize("rel", ["token", "table"])
@pytest.mark.parametrize("rel_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("extent,width", [(0, 0), (1, 1), (17, 40), (128, 128), (1024, 1025)])
def test_sparse_biases(cuda, rel, rel_dtype, extent, width):
    c = Sparse([70, 1, 9], [700, 40, 1200], 20, rel=rel, rel_dtype=rel_dtype, extent=extent,
               width=width, seed=extent)
    c.check(run(c, cuda))


@pytest.mark.parametrize("top", [1, 2, 3, 33, 64, 65, 150])
@pytest.mark.parametrize("kv", [None, F8])
@pytest.mark.parametrize("block", [8, 16, 128])
def test_sparse_lists(cuda, top, kv, block):
    """Short and long lists, more entries than blocks, shares of a list."""
    c = Sparse([1, 1, 3], [2000, 100, 3500], top, block=block, kv=kv, seed=top)
    c.check(run(c, cuda))


@pytest.mark.parametrize("d,block", [(64, 16), (64, 32), (128, 16)])
@pytest.mark.parametrize("kv", [None, F8])
@pytest.mark.parametrize("window", [0, 5, 30, 100, 500, 2 ** 31 - 1])
def test_sparse_windows(cuda, window, kv, d, block):
    c = Sparse(NEWS, LENS, 12, window=window, kv=kv, d=d, block=block, seed=window % 97)
    c.check(run(c, cuda))


@pytest.mark.parametrize("batch", [1, 2, 40, 130])
def test_sparse_steps(cuda, batch):
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(1, 3000, (batch,), generator=g).tolist()
    c = Sparse([1] * batch, lens, 32, seed=batch)
    c.check(run(c, cuda), seqs=set(range(min(batch, 20))) | {batch - 1})


def test_sparse_edges(cuda):
    """Tokens before the first key, empty lists, empty sequences, entries outside the pool."""
    for kv in (None, F8):
        c = Sparse([5, 140, 3, 0, 1, 4], [3, 64, 0, 0, 0, 300], 4, kv=kv, seed=5)
        c.check(run(c, cuda))
        c.lists[:] = -1
        out, lse = run(c, cuda)
        assert not out.any() and lse.isneginf().all()
        c = Sparse(NEWS, LENS, 9, kv=kv, seed=8)
        c.table[3, 4], c.table[4, 0], c.table[6, 12], c.table[8, 100] = -1, 1 << 20, -(1 << 31), c.kc.shape[0]
        c.check(run(c, cuda))
    c = Sparse([0, 0], [20, 30])
    out, lse = run(c, cuda)
    assert out.shape == (0, 8, 128) and lse.shape == (8, 0)


@pytest.mark.parametrize("kv", [None, F8])
def test_sparse_reads_no_other_block(cuda, kv):
    """Blocks that no list names, rows past the last key and rows left of the window may hold NaN."""
    c = Sparse([1, 3], [1000, 777], 9, kv=kv, window=600, seed=9)
    clean = c.kc, c.vc
    keep = torch.zeros(c.kc.shape[:2], dtype=torch.bool)
    t = 0
    for b, (n, lk) in enumerate(zip(c.news, c.lens)):
        for i in range(n):
            pos = lk - n + i
            for blk in set(c.lists[t].flatten().tolist()) - {-1}:
                rows = torch.arange(c.block) + blk * c.block
                keep[int(c.table[b, blk])] |= (rows <= pos) & (rows >= pos - 600)
            t += 1
    c.kc, c.vc = (torch.where(keep[..., None, None], x.float(), math.nan).to(x.dtype) for x in clean)
    got = run(c, cuda)
    c.kc, c.vc = (torch.nan_to_num(x.float(), 0.0).to(x.dtype) for x in (c.kc, c.vc))
    c.check(got)


# Many tokens.


@pytest.mark.parametrize("hq,hkv,d,dtype,block", [
    (8, 2, 128, torch.bfloat16, 16), (8, 2, 64, torch.float16, 16), (4, 4, 64, torch.bfloat16, 8),
    (8, 1, 128, torch.float16, 32), (6, 2, 128, torch.bfloat16, 8), (10, 2, 64, torch.float16, 64),
    (4, 2, 128, torch.bfloat16, 256), (7, 1, 128, torch.bfloat16, 16)])
@pytest.mark.parametrize("kv", [None, F8])
@pytest.mark.parametrize("messy", [False, True])
def test_sparse_many_tokens(cuda, hq, hkv, d, dtype, block, kv, messy):
    if kv and block * d < 1024:
        pytest.skip("e4m3 blocks of one load at least")
    news = [1400, 3, 700] if hkv > 2 else [900, 3, 170] if hkv > 1 else [530, 3, 40]
    c = Sparse(news, [1500, 70, 2300], 9, messy, hq=hq, hkv=hkv, d=d, dtype=dtype, block=block, kv=kv,
               extent=50, seed=hq + d + block)
    c.check(run(c, cuda))


@pytest.mark.parametrize("top", [1, 2, 40, 129, 512])
@pytest.mark.parametrize("kv", [None, F8])
def test_sparse_many_tokens_lists(cuda, top, kv):
    c = Sparse([600, 0, 600], [1700, 9, 600], top, kv=kv, window=300 if top == 40 else -1, seed=top)
    c.check(run(c, cuda))


@pytest.mark.parametrize("kv", [None, F8])
def test_sparse_many_tokens_that_list_alike(cuda, kv):
    """All tokens the same blocks, one of them many times over."""
    c = Sparse([1100], [1900], 20, kv=kv, seed=22)
    c.lists[:] = torch.randint(0, 60, (20,), generator=torch.Generator().manual_seed(22)).to(torch.int32)
    c.lists[500:, :, 3:9] = 7
    c.check(run(c, cuda))
    again = run(c, cuda)
    assert all(torch.equal(a, b) for a, b in zip(again, run(c, cuda)))


def test_sparse_many_tokens_edges(cuda):
    """Tokens before the first key or with empty lists, entries outside the pool, other strides."""
    c = Sparse([900, 200, 1], [500, 200, 40], 9, messy=True, seed=23)
    c.table[0, 4], c.table[1, 3], c.table[1, 5] = -1, 1 << 20, c.kc.shape[0]
    c.lists[300:420] = -1
    c.check(run(c, cuda))
    wide = torch.full((c.lists.shape[0], 3, 20), 5, dtype=torch.int32)
    wide[:, 1:, 7:16] = c.lists
    c.check(run(c, cuda, lists=wide.to(cuda)[:, 1:, 7:16]))


@pytest.mark.parametrize("kv", [None, F8])
def test_sparse_many_tokens_read_no_other_block(cuda, kv):
    """Blocks that no list names, rows past the last key and rows left of the windows may hold NaN,
    and a block that only a neighbour lists."""
    c = Sparse([1040], [1600], 9, kv=kv, window=700, seed=24)
    clean = c.kc, c.vc
    c.lists[:, :, :4] = torch.randint(36, 60, (4,), generator=torch.Generator().manual_seed(24)).to(torch.int32)
    c.lists[(c.lists >= 60) & (c.lists < 90)] = -1
    keep = torch.zeros(c.kc.shape[:2], dtype=torch.bool)
    for i in range(1040):
        pos = 560 + i
        for blk in set(c.lists[i].flatten().tolist()) - {-1}:
            rows = torch.arange(c.block) + blk * c.block
            keep[int(c.table[0, blk])] |= (rows <= pos) & (rows >= pos - 700)
    assert not keep[c.table[0, 60:90].long()].any()
    c.kc, c.vc = (torch.where(keep[..., None, None], x.float(), math.nan).to(x.dtype) for x in clean)
    got = run(c, cuda)
    c.kc, c.vc = (torch.nan_to_num(x.float(), 0.0).to(x.dtype) for x in (c.kc, c.vc))
    c.check(got)
    # a block of NaN costs the tokens that list it, no other
    c.kc[int(c.table[0, 70])] = c.vc[int(c.table[0, 70])] = math.nan
    c.lists = c.lists.clone()
    c.lists[600:900:7, :, 5] = 70
    out, lse = run(c, cuda)
    hit = torch.zeros(1040, dtype=torch.bool)
    hit[600:900:7] = True
    assert not out[~hit].isnan().any() and not lse[:, ~hit].isnan().any()


@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.bfloat16).min])
@pytest.mark.parametrize("news,lens", [([70, 1, 9], [200, 40, 60]), ([1, 1, 1], [900, 40, 5])])
def test_biases_that_hide_keys(cuda, low, news, lens):
    """-inf, and the type's lowest value, whose quotient by the scale leaves fp32: the key is hidden;
    a row whose bias hides all of its keys is empty.  Listed blocks and the whole cache alike."""
    c = Sparse(news, lens, 130, extent=64, seed=25)
    c.lists = torch.arange(130, dtype=torch.int32).expand(sum(news), c.hkv, 130).contiguous()
    g = torch.Generator().manual_seed(25)
    c.rel[torch.rand(c.rel.shape, generator=g) < 0.3] = low
    c.rel[-1] = low
    args, lists = c.on(cuda), c.lists.to(cuda)
    got = [x.cpu() for x in inkling_fa4_rel_attention_sparse_paged(*args, lists, c.max_q, c.max_k,
                                                                   c.extent, **c.settings())]
    whole = [x.cpu() for x in inkling_fa4_rel_attention_paged(*args, c.max_q, c.max_k, c.extent,
                                                              **c.settings())]
    c.rel[c.rel == low] = -math.inf
    for out, lse in (got, whole):
        assert not out.isnan().any() and not lse.isnan().any()
        c.check((out, lse))
    if lens[-1] <= 64:
        assert not got[0][-1].any() and got[1][:, -1].isneginf().all()


@pytest.mark.parametrize("layout", ["heads", "joint"])
@pytest.mark.parametrize("kv", [None, F8])
def test_sparse_layouts(cuda, layout, kv):
    c = Sparse(NEWS, LENS, 8, layout=layout, kv=kv, seed=6)
    c.check(run(c, cuda))


@pytest.mark.parametrize("news,lens", [(NEWS, LENS), ([1, 1, 1], [900, 2000, 5])])
@pytest.mark.parametrize("kv", [None, F8])
def test_sparse_over_all_blocks_is_the_attention(cuda, news, lens, kv):
    c = Sparse(news, lens, 130, kv=kv, seed=10)
    c.lists = torch.arange(130, dtype=torch.int32).expand(sum(news), c.hkv, 130).contiguous()
    # the two round each weight to 16 bits relative to bases of their own, so they differ by up
    # to twice the bound that each keeps to the definition
    c.check(run(c, cuda))
    want = inkling_fa4_rel_attention_paged(*c.on(cuda), c.max_q, c.max_k, c.extent, **c.settings())
    c.check([x.cpu() for x in want])


def test_sparse_strided_lists(cuda):
    c = Sparse(NEWS, LENS, 8, seed=11)
    wide = torch.full((c.lists.shape[0], 3, 20), 5, dtype=torch.int32)
    wide[:, 1:, 7:15] = c.lists
    c.check(run(c, cuda, lists=wide.to(cuda)[:, 1:, 7:15]))
    one = c.lists[:1].expand(c.lists.shape)  # one list for all tokens
    c.lists = one
    c.check(run(c, cuda, lists=one[:1].to(cuda).expand(one.shape)))


def test_sparse_far_blocks(cuda):
    """A pool of more than 2^32 elements."""
    c = Sparse([2, 9], [200, 90], 5, seed=13)
    args = c.on(cuda)
    blocks = (1 << 32) // (c.block * c.hkv * c.d) + 64
    far = c.table.clone()
    high = torch.arange(c.table.shape[1]) % 2 == 0
    far[:, high] = torch.where(c.table < c.kc.shape[0], far + blocks - c.kc.shape[0], far)[:, high]
    for i in (1, 2):
        pool = torch.empty((blocks,) + args[i].shape[1:], dtype=args[i].dtype, device=cuda)
        pool[:c.kc.shape[0]] = args[i]
        pool[-c.kc.shape[0]:] = args[i]
        args[i] = pool
    args[6] = far.to(cuda)
    out, lse = inkling_fa4_rel_attention_sparse_paged(*args, c.lists.to(cuda), c.max_q, c.max_k,
                                                      c.extent, **c.settings())
    bounds = torch.zeros(blocks, c.hkv, 2, c.d, device=cuda).bfloat16()
    inkling_fa4_key_bounds_paged(args[1], bounds, *args[4:], c.max_q)
    torch.cuda.synchronize()
    c.check((out.cpu(), lse.cpu()))
    want = want_bounds(c, torch.zeros(c.kc.shape[0], c.hkv, 2, c.d).bfloat16())
    for b in range(2):
        for blk in range((c.lens[b] - c.news[b]) // 16, -(-c.lens[b] // 16)):
            assert torch.equal(bounds[int(far[b, blk])].cpu(), want[int(c.table[b, blk])])


def test_sparse_rows_of_no_sequence(cuda):
    for news, lens, top in (([5, 9], [50, 60], 4), ([1, 1], [900, 2000], 60)):
        c = Sparse(news, lens, top, seed=18)
        n = sum(news)
        args = c.on(cuda)
        args[0] = torch.cat([args[0], args[0][:2]])
        args[3] = torch.cat([args[3], args[3][:2]])
        lists = torch.cat([c.lists, c.lists[:2]]).to(cuda)
        torch.use_deterministic_algorithms(True)
        try:
            out, lse = inkling_fa4_rel_attention_sparse_paged(*args, lists, c.max_q, c.max_k,
                                                              c.extent, **c.settings())
        finally:
            torch.use_deterministic_algorithms(False)
        torch.cuda.synchronize()
        assert out[n:].isnan().all() and lse[:, n:].isnan().all()
        c.check((out[:n].cpu(), lse[:, :n].cpu()))


def test_sparse_refusals(cuda):
    c = Sparse([3, 4], [40, 50], seed=19)
    args = c.on(cuda) + [c.lists.to(cuda)]

    def call(i=None, x=None, extent=c.extent, max_k=c.max_k, **kw):
        a = list(args)
        if i is not None:
            a[i] = x
        return inkling_fa4_rel_attention_sparse_paged(*a, c.max_q, max_k, extent,
                                                      **dict(c.settings(), **kw))

    q, kc, vc, rel, cu, used, table, lists = args
    for i, bad in [(0, q.float()), (0, q[:, :7]), (1, kc[0]), (1, kc.half()), (2, vc[:-1]),
                   (3, rel[:-1]), (4, cu.long()), (5, used[:1]), (6, table.long()), (7, lists.long()),
                   (7, lists[:-1]), (7, lists[:, :1]), (7, lists[:, :, :0]), (7, lists[:, :, ::2]),
                   (7, lists.cpu()), (7, lists[0])]:
        with pytest.raises((ValueError, RuntimeError, IndexError)):
            call(i, bad)
    for kw in (dict(extent=c.extent + 1), dict(softmax_scale=math.nan), dict(max_k=1 << 20)):
        with pytest.raises((ValueError, RuntimeError)):
            call(**kw)
    wide = Sparse([3], [40], hq=17, hkv=1)
    with pytest.raises(RuntimeError, match="EUNSUPPORTED"):
        run(wide, cuda)
    torch.cuda.synchronize()


# ---- together ------------------------------------------------------------------------------------


@pytest.mark.parametrize("kv", [None, F8])
def test_a_prompt_in_chunks_then_steps(cuda, kv):
    """Append, bounds, choice and attention, chunk by chunk and token by token, one captured step
    replayed; against the definitions on what the cache holds."""
    g = torch.Generator().manual_seed(20)
    batch, hq, hkv, d, block, extent, top = 3, 8, 2, 128, 16, 64, 6
    pool, cap = 100, 30
    scale = 0.02 if kv else 1.0
    kc, vc = (torch.zeros(pool, block, hkv, d, device=cuda).to(kv or torch.bfloat16) for _ in range(2))
    bounds = torch.full((pool, hkv, 2, d), math.nan, device=cuda).to(kc.dtype)
    table = torch.randperm(pool, generator=g)[:batch * cap].view(batch, cap).to(torch.int32).to(cuda)
    held = [0] * batch
    quant = dict(k_scale=scale, v_scale=scale)

    def step(q, k, v, rel, cu, used, max_q, max_k):
        inkling_fa4_kv_append_paged(k, v, kc, vc, cu, used, table, **quant)
        inkling_fa4_key_bounds_paged(kc, bounds, cu, used, table, max_q)
        lists = inkling_fa4_select_blocks_paged(q, bounds, cu, used, table, block, max_q, max_k, top)
        out, lse = inkling_fa4_rel_attention_sparse_paged(
            q, kc, vc, rel, cu, used, table, lists, max_q, max_k, extent, softmax_scale=0.09,
            return_lse=True, **quant)
        return lists, out, lse

    def tokens(news):
        n = sum(news)
        x = [torch.randn(n, h, d, generator=g).bfloat16() for h in (hq, hkv, hkv)]
        return x + [(0.5 * torch.randn(n, hq, extent, generator=g)).bfloat16()]

    def check(news, q, rel, lists, out, lse):
        c = Sparse(news, held, top, hq=hq, hkv=hkv, d=d, kv=kv, extent=extent, scale=0.09)
        c.q, c.rel, c.table, c.scales = q, rel, table.cpu(), (scale, scale)
        c.kc, c.vc, c.lists = kc.cpu(), vc.cpu(), lists.cpu()
        assert torch.equal(c.lists, want_lists(c, bounds.cpu(), top, 1, 2))
        for b, lk in enumerate(held):  # the bounds are those of the whole cache
            for blk in range(-(-lk // block)):
                ent = int(c.table[b, blk])
                rows = c.kc[ent, :min(block, lk - blk * block)].float()
                assert same(bounds[ent, :, 0].cpu(), rows.amin(0)) and same(bounds[ent, :, 1].cpu(), rows.amax(0))
        c.check((out.cpu(), lse.cpu()))

    for news in ([100, 3, 40], [150, 200, 0], [1, 1, 1]):
        held = [a + b for a, b in zip(held, news)]
        q, k, v, rel = tokens(news)
        cu = torch.tensor([0] + news, dtype=torch.int32).cumsum(0).to(torch.int32).to(cuda)
        used = torch.tensor(held, dtype=torch.int32, device=cuda)
        got = step(q.to(cuda), k.to(cuda), v.to(cuda), rel.to(cuda), cu, used, max(news), max(held))
        torch.cuda.synchronize()
        check(news, q, rel, *got)
    # one captured decode step
    news = [1, 1, 1]
    ins = [x.to(cuda) for x in tokens(news)]
    cu = torch.arange(4, dtype=torch.int32, device=cuda)
    used = torch.tensor(held, dtype=torch.int32, device=cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*ins, cu, used, 1, cap * block)
    for _ in range(3):
        held = [a + 1 for a in held]
        new = tokens(news)
        for x, y in zip(ins, new):
            x.copy_(y)
        used.copy_(torch.tensor(held, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        check(news, new[0], new[3], *got)


def test_streams(cuda):
    c = Sparse([1, 1, 40], [900, 2000, 500], 30, seed=21)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        args = c.on(cuda)
        bounds = key_like_bounds(c).to(cuda)
        inkling_fa4_key_bounds_paged(args[1], bounds, *args[4:], c.max_q)
        lists = inkling_fa4_select_blocks_paged(args[0], bounds, *args[4:], 16, c.max_q, c.max_k, 30)
        out, lse = inkling_fa4_rel_attention_sparse_paged(*args, lists, c.max_q, c.max_k, c.extent,
                                                          **c.settings())
        got = bounds.cpu(), lists.cpu(), out.cpu(), lse.cpu()
    assert same(got[0], want_bounds(c, key_like_bounds(c)))
    c.lists = got[1]
    assert torch.equal(c.lists, want_lists(c, got[0], 30, 1, 2))
    c.check(got[2:])
