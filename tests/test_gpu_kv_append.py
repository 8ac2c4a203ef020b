"""Paged append on the GPU: the written rows against the fp64 oracle, every other row
untouched, and bad lengths and pages (bounds: tests/test_gpu_norm_rope.py; an e4m3 row
carries half an e4m3 step, 2^-4 of the value and 2^-10 below its normal range, more)."""
import math

import pytest
import torch

from inkling_fa4 import (inkling_fa4_kv_append_paged, inkling_fa4_qk_norm_rope,
                         inkling_fa4_rel_attention, inkling_fa4_rel_attention_decode_paged)
from oracle import ref_rel_attn_paged_with_lse
from oracle.norm_rope import append_positions, norm_rope

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-6
F8 = torch.float8_e4m3fn


class Call:
    """An append of `new` tokens behind `past` keys per sequence, on a pool of random rows."""

    def __init__(self, new, past, hq=4, hkv=2, d=64, dtype=torch.bfloat16, kv=None, block=16,
                 rot=32, normed=True, seed=0, tail=0):
        g = torch.Generator().manual_seed(seed)
        self.new, self.past, self.block, self.hq, self.hkv = new, past, block, hq, hkv
        tokens = sum(new) + tail
        x = torch.randn(tokens, hq + 2 * hkv, d, generator=g).to(dtype)
        self.q, self.k, self.v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
        w = [(1 + 0.2 * torch.randn(d, generator=g)) for _ in range(2)]
        self.qw, self.kw = w if normed else (None, None)
        used = [a + b for a, b in zip(new, past)]
        need = [max(1, -(-n // block)) for n in used]
        order = torch.randperm(sum(need) + 3, generator=g).to(torch.int32)
        self.table = torch.full((len(new), max(need, default=1)), 1 << 30, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.cu = torch.tensor([0] + [sum(new[:i + 1]) for i in range(len(new))], dtype=torch.int32)
        self.used = torch.tensor(used, dtype=torch.int32)
        pool = (sum(need) + 3, block, hkv, d)
        self.kc, self.vc = (torch.randn(*pool, generator=g).to(kv or dtype) for _ in range(2))
        angle = 6.3 * torch.rand(max(used, default=0) + 1, rot // 2, generator=g)
        self.cos, self.sin = (angle.cos(), angle.sin()) if rot else (None, None)

    def run(self, dev, q=True, **kw):
        def on(t):
            return None if t is None else t.to(dev)
        print(f"append: new {self.new[:6]} past {self.past[:6]} heads {self.hq}/{self.hkv} "
              f"pool {tuple(self.kc.shape)} {self.kc.dtype} {kw}", flush=True)
        kc, vc = on(self.kc), on(self.vc)
        whole = torch.cat([self.q, self.k, self.v], 1).to(dev)
        out = inkling_fa4_kv_append_paged(
            whole[:, self.hq:self.hq + self.hkv], whole[:, self.hq + self.hkv:], kc, vc,
            on(self.cu), on(self.used), on(self.table), q=whole[:, :self.hq] if q else None,
            q_weight=on(self.qw) if q else None, k_weight=on(self.kw), cos=on(self.cos),
            sin=on(self.sin), eps=EPS, **kw)
        torch.cuda.synchronize()
        return out, kc.cpu(), vc.cpu()

    def slots(self):
        """(token, position, block, row) of the tokens that are written."""
        for t, b, p in append_positions(self.cu, self.used):
            if 0 <= p < self.table.shape[1] * self.block:
                blk = int(self.table[b, p // self.block])
                if 0 <= blk < self.kc.shape[0]:
                    yield t, p, blk, p % self.block

    def check(self, got, k_scale=1.0, v_scale=1.0, interleaved=False):
        out, kc, vc = got
        rows = list(self.slots())
        t, p, blk, row = (torch.tensor(x, dtype=torch.long) for x in zip(*rows))
        cs, sn = (None, None) if self.cos is None else (self.cos[p], self.sin[p])
        want, size = norm_rope(self.k[t], self.kw, cs, sn, EPS, interleaved)
        _near(kc[blk, row], want / k_scale, 40 * U * size / k_scale)
        if kc.dtype == F8:
            _near(vc[blk, row], self.v[t].double() / v_scale, U * self.v[t].double().abs() / v_scale)
        else:
            assert torch.equal(vc[blk, row], self.v[t])
        if out is not None:
            want, size = norm_rope(self.q[t], self.qw, cs, sn, EPS, interleaved)
            _near(out.cpu()[t], want, 40 * U * size)
        keep = torch.ones(kc.shape[:2], dtype=torch.bool)
        keep[blk, row] = False
        for a, b in ((kc, self.kc), (vc, self.vc)):
            assert torch.equal(a.view(torch.uint8)[keep], b.view(torch.uint8)[keep])


def _near(got, want, slack):
    if got.dtype == F8:
        want = want.clamp(-448, 448)
        bound = 2.0 ** -4 * (want.abs() + slack) + slack + 2.0 ** -10
    else:
        i = torch.finfo(got.dtype)
        bound = i.eps / 2 * (want.abs() + slack) + slack + i.tiny * i.eps
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), float((got.double() - want).abs().max()))


@pytest.mark.parametrize("kv", [None, F8])
@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("block", [8, 16, 128])
def test_decode_step(cuda, d, block, kv):
    past = [0, 1, 7, 8, 15, 16, 31, 127, 128, 300]
    c = Call([1] * len(past), past, 8, 2, d, kv=kv, block=block, rot=d, seed=block + d)
    s = dict(k_scale=0.031, v_scale=0.07) if kv else {}
    c.check(c.run(cuda, **s), **s)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kv", [None, F8])
def test_ragged_chunks(cuda, kv, dtype, interleaved):
    """Sequences without new tokens between others, a first chunk, chunks that cross pages."""
    c = Call([0, 5, 0, 0, 70, 1, 33, 0], [9, 0, 0, 40, 11, 16, 100, 3], dtype=dtype, kv=kv, seed=3)
    s = dict(k_scale=1 / 64, v_scale=1 / 32) if kv else {}
    c.check(c.run(cuda, interleaved=interleaved, **s), interleaved=interleaved, **s)


@pytest.mark.parametrize("batch", [1, 2, 16, 17, 64, 257, 1025])
def test_batches(cuda, batch):
    """The search for a token's sequence: one to three rounds, with and without empty ones."""
    g = torch.Generator().manual_seed(batch)
    new = [int(x) for x in torch.randint(0, 4, (batch,), generator=g)]
    new[0] = max(new[0], 1)
    past = [int(x) for x in torch.randint(0, 40, (batch,), generator=g)]
    for d in (64, 128):
        c = Call(new, past, 2, 1, d, rot=16, seed=batch)
        c.check(c.run(cuda))


def test_rotation_only_norm_only_and_neither(cuda):
    for rot, normed in ((64, False), (0, True), (0, False)):
        c = Call([3, 1], [14, 2], rot=rot, normed=normed, seed=5)
        c.check(c.run(cuda))


def test_without_queries(cuda):
    c = Call([3, 20], [14, 2], seed=6)
    got = c.run(cuda, q=False)
    assert got[0] is None
    c.check(got)
    # the queries' launch writes the same rows
    again = c.run(cuda)
    assert torch.equal(got[1], again[1]) and torch.equal(got[2], again[2])


def test_lengths_and_pages_outside_the_contract(cuda):
    """More new tokens than keys (negative positions), a length past the table, entries outside
    the pool, tokens behind the last sequence: those rows are not written, all others are."""
    c = Call([5, 4, 6, 2], [20, 30, 10, 0], seed=7, tail=3)
    c.used[0] = 3           # positions -2 .. 2
    c.used[1] = c.table.shape[1] * c.block + 2  # two positions past the table
    c.table[2, 0] = -1
    c.table[3, 0] = c.kc.shape[0]
    c.cos, c.sin = c.cos.repeat(3, 1), c.sin.repeat(3, 1)
    c.check(c.run(cuda))


def test_offsets_that_decrease_or_leave_the_tensors(cuda):
    """cu_seqlens that break their contract write unspecified rows of the pool at most: the
    call returns, and nothing outside the pool's sequences changes."""
    c = Call([4, 4, 4], [10, 20, 30], seed=8)
    for cu in ([0, 9, 3, 12], [5, 4, 3, 2], [0, 4, 8, 1 << 30], [-7, 4, 8, 12], [3, 3, 3, 3]):
        c.cu = torch.tensor(cu, dtype=torch.int32)
        _, kc, vc = c.run(cuda)
        owned = torch.zeros(kc.shape[0], dtype=torch.bool)
        for b in range(3):
            n = -(-int(c.used[b]) // c.block)
            owned[c.table[b, :n].long()] = True
        for a, b in ((kc, c.kc), (vc, c.vc)):
            assert torch.equal(a[~owned], b[~owned])


def test_empty_calls(cuda):
    c = Call([0, 0], [5, 9], seed=9)
    out, kc, vc = c.run(cuda)
    assert out.shape[0] == 0 and torch.equal(kc, c.kc) and torch.equal(vc, c.vc)
    c = Call([], [], seed=9, tail=2)
    _, kc, vc = c.run(cuda)
    assert torch.equal(kc, c.kc) and torch.equal(vc, c.vc)


def test_fp8_rounding_saturation_and_nan(cuda):
    """v alone (no arithmetic but the scale): nearest even, +-448 past the range, NaN stays."""
    c = Call([1], [0], 0 + 1, 1, 64, kv=F8, rot=0, normed=False, seed=1)
    x = torch.tensor([0.0, -0.0, 17.0, 19.0, 447.0, 464.0, 1e4, -1e4, math.inf, -math.inf, 2 ** -9,
                      2 ** -10, 1.5 * 2 ** -9, -17.0, 1.0625, 1.1875] * 4).to(torch.bfloat16)
    x[37] = math.nan
    c.v = x.view(1, 1, 64).clone()
    _, _, vc = c.run(cuda)
    got = vc[int(c.table[0, 0]), 0, 0].float()
    want = x.float().clamp(-448, 448).to(F8).float()
    assert torch.equal(got.nan_to_num(99.0), want.nan_to_num(99.0)) and got[37].isnan()


def test_blocks_past_32_bits_of_elements(cuda):
    """The same blocks at the end of a pool of 2^32 elements and more: the same rows there."""
    c = Call([20, 1, 33], [5, 70, 0], d=128, seed=19)
    want = c.run(cuda)
    few = c.kc.shape[0]
    shift = (1 << 32) // c.kc[0].numel() + 1000 - few
    pools = []
    for x in (c.kc, c.vc):
        big = torch.empty(shift + few, *x.shape[1:], dtype=x.dtype, device=cuda)
        big[shift:] = x.to(cuda)
        pools.append(big)
    table = torch.where(c.table < few, c.table + shift, c.table).to(cuda)
    on = [x.to(cuda) for x in (c.cu, c.used)]
    q = inkling_fa4_kv_append_paged(
        c.k.to(cuda), c.v.to(cuda), *pools, *on, table, q=c.q.to(cuda), q_weight=c.qw.to(cuda),
        k_weight=c.kw.to(cuda), cos=c.cos.to(cuda), sin=c.sin.to(cuda), eps=EPS)
    assert torch.equal(q, want[0])
    for big, x in zip(pools, want[1:]):
        assert torch.equal(big[shift:].cpu(), x)


def test_strided_caches(cuda):
    """A pool that keeps k and v of a block side by side, and one with the heads outermost."""
    c = Call([3, 18], [14, 2], seed=10)
    want = c.run(cuda)
    n, bs, hkv, d = c.kc.shape
    both = torch.stack([c.kc, c.vc], 1).to(cuda)
    first = torch.stack([c.kc.permute(0, 2, 1, 3), c.vc.permute(0, 2, 1, 3)]).to(cuda)
    for kc, vc in ((both[:, 0], both[:, 1]), (first[0].transpose(1, 2), first[1].transpose(1, 2))):
        inkling_fa4_kv_append_paged(c.k.to(cuda), c.v.to(cuda), kc, vc, c.cu.to(cuda),
                                    c.used.to(cuda), c.table.to(cuda), k_weight=c.kw.to(cuda),
                                    cos=c.cos.to(cuda), sin=c.sin.to(cuda), eps=EPS)
        torch.cuda.synchronize()
        assert torch.equal(kc.cpu(), want[1]) and torch.equal(vc.cpu(), want[2])


def test_same_rows_as_the_norm_operator(cuda):
    """k and q of an append are, bit by bit, those of inkling_fa4_qk_norm_rope."""
    c = Call([9, 4], [10, 3], 8, 2, 128, rot=128, seed=12)
    out, kc, _ = c.run(cuda)
    pos = torch.tensor([p for _, p, _, _ in c.slots()], dtype=torch.int32)
    q, k = inkling_fa4_qk_norm_rope(*(x.to(cuda) for x in (c.q, c.k, c.qw, c.kw, c.cos, c.sin, pos)),
                                    eps=EPS)
    assert torch.equal(out, q)
    for t, _, blk, row in c.slots():
        assert torch.equal(kc[blk, row], k[t].cpu())


def test_graph_replays(cuda):
    """A captured append writes where the lengths and tables then say."""
    c = Call([1] * 6, [3, 15, 16, 40, 0, 9], seed=13)
    k, v, kc, vc, cu, used, table, q = (x.to(cuda) for x in (
        c.k, c.v, c.kc, c.vc, c.cu, c.used, c.table, c.q))
    kw, qw, cos, sin = (x.to(cuda) for x in (c.kw, c.qw, c.cos.repeat(2, 1), c.sin.repeat(2, 1)))

    def step(kc, vc):
        return inkling_fa4_kv_append_paged(k, v, kc, vc, cu, used, table, q=q, q_weight=qw,
                                           k_weight=kw, cos=cos, sin=sin)
    step(kc.clone(), vc.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(kc, vc)
    ke, ve = kc.clone(), vc.clone()
    for i in range(4):
        k.normal_()
        v.normal_()
        q.normal_()
        used.copy_((c.used - i).clamp(min=1).to(cuda))
        graph.replay()
        want = step(ke, ve)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(kc, ke) and torch.equal(vc, ve)


def test_prefill_decode_steps_through_the_cache(cuda):
    """Chunks appended, then decode steps: append and attention over the pages, against the
    oracle on the oracle's own keys (out 2e-2: keys and queries differ from the oracle's by
    16-bit rounding, as in the paged decode tests)."""
    lens, steps, hq, hkv, d = [40, 7, 129], 3, 8, 2, 128
    total = [n + steps for n in lens]
    c = Call(total, [0, 0, 0], hq, hkv, d, rot=64, seed=14)
    kc, vc, table = c.kc.to(cuda), c.vc.to(cuda), c.table.to(cuda)
    w = [x.to(cuda) for x in (c.qw, c.kw, c.cos, c.sin)]
    start = c.cu.tolist()
    gen = torch.Generator().manual_seed(15)
    rel = 0.5 * torch.randn(3, hq, 64, generator=gen)

    def append(first, count):
        rows = torch.cat([torch.arange(start[b] + first[b], start[b] + first[b] + count[b])
                          for b in range(3)])
        cu = torch.tensor([0] + [sum(count[:i + 1]) for i in range(3)], dtype=torch.int32)
        used = torch.tensor([f + n for f, n in zip(first, count)], dtype=torch.int32).to(cuda)
        q = inkling_fa4_kv_append_paged(c.k[rows].to(cuda), c.v[rows].to(cuda), kc, vc, cu.to(cuda),
                                        used, table, q=c.q[rows].to(cuda), q_weight=w[0],
                                        k_weight=w[1], cos=w[2], sin=w[3], eps=EPS)
        return q, used, rows
    append([0, 0, 0], lens)
    for i in range(steps):
        q, used, rows = append([n + i for n in lens], [1, 1, 1])
        cu = torch.arange(4, dtype=torch.int32)
        out = inkling_fa4_rel_attention_decode_paged(
            q, kc, vc, rel.to(cuda), cu.to(cuda), used, table, 1, max(total), 64,
            softmax_scale=0.1, bottom_right=True)
        torch.cuda.synchronize()
        pos = torch.tensor([n + i for n in lens])
        qo = norm_rope(c.q[rows], c.qw, c.cos[pos], c.sin[pos], EPS)[0].to(torch.bfloat16)
        ko, vo = c.kc.clone(), c.vc.clone()
        for t, p, blk, row in c.slots():
            ko[blk, row] = norm_rope(c.k[t:t + 1], c.kw, c.cos[p:p + 1], c.sin[p:p + 1],
                                     EPS)[0][0].to(torch.bfloat16)
            vo[blk, row] = c.v[t]
        want, _ = ref_rel_attn_paged_with_lse(qo, ko, vo, rel, cu, used.cpu(), c.table, 0.1, 64,
                                              bottom_right=True)
        torch.testing.assert_close(out.float().cpu(), want.float(), atol=2e-2, rtol=2e-2)


def test_refusals(cuda):
    c = Call([2, 1], [3, 4], seed=16)
    ok = dict(k=c.k, v=c.v, k_cache=c.kc, v_cache=c.vc, cu_seqlens_q=c.cu, seqused_k=c.used,
              block_table=c.table, q=c.q, q_weight=c.qw, k_weight=c.kw, cos=c.cos, sin=c.sin)
    ok = {n: x.to(cuda) for n, x in ok.items()}
    inkling_fa4_kv_append_paged(**ok)
    kc = ok["k_cache"]
    for bad in (dict(v=ok["v"][:1]), dict(v=ok["v"][:, :1]), dict(k=ok["k"].float()),
                dict(k_cache=kc[0]), dict(k_cache=kc[:, :, :1]), dict(k_cache=kc.half()),
                dict(k_cache=kc.to(F8)), dict(k_cache=kc[..., ::2], v_cache=kc[..., ::2]),
                dict(k_cache=kc[:, :12], v_cache=kc[:, :12]),
                dict(k_cache=kc.cpu()), dict(cu_seqlens_q=ok["cu_seqlens_q"].long()),
                dict(cu_seqlens_q=ok["cu_seqlens_q"][:2]), dict(seqused_k=ok["seqused_k"][:1]),
                dict(block_table=ok["block_table"][:1]), dict(block_table=ok["block_table"].t()),
                dict(block_table=ok["block_table"].long()), dict(q=ok["q"][:2]), dict(q=None),
                dict(sin=None), dict(cos=ok["cos"].half(), sin=ok["sin"].half()),
                dict(k_cache=kc.to(F8), v_cache=kc.to(F8), k_scale=0.0),
                dict(k_cache=kc.to(F8), v_cache=kc.to(F8), v_scale=math.nan),
                dict(k_cache=kc[:1].expand(4, -1, -1, -1), v_cache=kc[:1].expand(4, -1, -1, -1))):
        with pytest.raises(RuntimeError):
            inkling_fa4_kv_append_paged(**dict(ok, **bad))


def test_no_gradient_is_asked_of_the_result(cuda):
    c = Call([1], [4], seed=17)
    q = c.q.to(cuda).requires_grad_()
    out = inkling_fa4_kv_append_paged(c.k.to(cuda), c.v.to(cuda), c.kc.to(cuda), c.vc.to(cuda),
                                      c.cu.to(cuda), c.used.to(cuda), c.table.to(cuda), q=q,
                                      q_weight=c.qw.to(cuda))
    assert not out.requires_grad


def test_strides_of_dimensions_of_one(cuda):
    """One token, one head, one block: their strides are never stepped along and say nothing."""
    c = Call([1], [3], 1, 1, seed=20)
    c.kc, c.vc = c.kc[:1], c.vc[:1]
    c.table[:] = 0
    want = c.run(cuda)
    q, k, v = (t.contiguous().to(cuda).as_strided((1, 1, 64), (67, 3, 1)) for t in (c.q, c.k, c.v))
    kc, vc = (t.clone().to(cuda).as_strided((1, 16, 1, 64), (7, 64, 3, 1)) for t in (c.kc, c.vc))
    out = inkling_fa4_kv_append_paged(k, v, kc, vc, c.cu.to(cuda), c.used.to(cuda), c.table.to(cuda),
                                      q=q, q_weight=c.qw.to(cuda), k_weight=c.kw.to(cuda),
                                      cos=c.cos.to(cuda), sin=c.sin.to(cuda), eps=EPS)
    assert torch.equal(out, want[0])
    assert torch.equal(kc.cpu(), want[1]) and torch.equal(vc.cpu(), want[2])


@pytest.mark.parametrize("scale", [7.0, 13.0, 0.03, 0.3, 1 / 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_fp8_of_every_16_bit_value(cuda, dtype, scale):
    """The e4m3 values of the fp32 quotients k / k_scale and v / v_scale, ties to even, whatever
    the scale (no norm, no rotation: rows go into the cache as they are)."""
    x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype)
    n = x.numel() // 64
    c = Call([n], [0], 0 + 1, 1, 64, dtype, kv=F8, rot=0, normed=False, seed=1)
    c.k = c.v = x.view(n, 1, 64).clone()
    _, kc, vc = c.run(cuda, k_scale=scale, v_scale=scale)
    want = (x.float() / torch.tensor(scale)).clamp(-448, 448).to(F8).float().view(n, 64)
    pages = c.table[0].long()
    for cache in (kc, vc):
        got = cache[pages].reshape(-1, 64)[:n].float()
        assert torch.equal(got.isnan(), want.isnan())
        off = (got != want) & ~want.isnan()
        assert not off.any(), (int(off.sum()), x.view(n, 64)[off][:3], got[off][:3], want[off][:3])


@pytest.mark.parametrize("kv", [None, F8])
def test_a_prompt_through_norm_attention_and_append(cuda, kv):
    """A prompt's three calls: norm and rotation, attention over what comes back, an append of that
    k as it is.  The cache holds, bit by bit, what the append's own norm and rotation write in
    16 bits; an e4m3 row is then the nearest of a 16-bit value.  A prompt's last row is that of a
    decode over the cache: 2e-2 apart at most, as in the decode tests (16-bit weights and outputs of
    two kernels), where the cache holds the same keys."""
    lens, hq, hkv, d = [40, 7, 129], 8, 2, 128
    c = Call(lens, [0, 0, 0], hq, hkv, d, kv=kv, rot=64, seed=21)
    q, k, v, qw, kw, cos, sin, cu, used, table = (x.to(cuda) for x in (
        c.q, c.k, c.v, c.qw, c.kw, c.cos, c.sin, c.cu, c.used, c.table))
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).to(cuda)
    kc, vc = c.kc.to(cuda), c.vc.to(cuda)
    q, k = inkling_fa4_qk_norm_rope(q, k, qw, kw, cos, sin, pos, eps=EPS)
    rel = (0.5 * torch.randn(sum(lens), hq, 64, generator=torch.Generator().manual_seed(22))).to(cuda)
    out = inkling_fa4_rel_attention(q, k, v, rel, cu, cu, max(lens), max(lens), 64, softmax_scale=0.1)
    scales = dict(k_scale=0.03, v_scale=0.02) if kv else {}
    assert inkling_fa4_kv_append_paged(k, v, kc, vc, cu, used, table, **scales) is None
    if kv:
        for cache, x, s in ((kc, k, 0.03), (vc, v, 0.02)):
            want = (x.float() / torch.tensor(s, device=cuda)).clamp(-448, 448).to(F8)
            for t, _, blk, row in c.slots():
                assert torch.equal(cache[blk, row].float(), want[t].float())
        return
    _, k2, v2 = c.run(cuda)
    assert torch.equal(kc.cpu(), k2) and torch.equal(vc.cpu(), v2)
    last = (cu[1:] - 1).long()
    got = inkling_fa4_rel_attention_decode_paged(
        q[last], kc, vc, rel[last].contiguous(), torch.arange(4, dtype=torch.int32, device=cuda), used,
        table, 1, max(lens), 64, softmax_scale=0.1, bottom_right=True)
    torch.testing.assert_close(got.float(), out[last].float(), atol=2e-2, rtol=2e-2)
