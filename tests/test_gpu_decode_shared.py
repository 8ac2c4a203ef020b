"""Decode behind a shared prefix on the GPU against the definition in fp64.

Bounds (u = 2^-24; h = half a step of q's type relative to the value; p the weights, n the keys):
  a score is off by at most ds = u ((D + 8) scale sum |q k| + 8 max|s|), the dot product of D
  exact products summed in fp32, its scaling, the bias and the maximum's subtraction; a weight
  by that, exp2's and the rounding to q's type, h; the sums add n u.  So
  out: h |out| + (h + 2 ds + (n + 64) u) A, A = sum p |v| / sum p, and in fp16, where weights
  below 2^-14 of the largest lose bits, 2^-25 sum |v|
  lse: ds + (n + 64) u + 8 u |lse|.
"""
import math

import pytest
import torch

from inkling_fa4 import (inkling_fa4_kv_append_paged,
                         inkling_fa4_rel_attention_decode_paged,
                         inkling_fa4_rel_attention_decode_shared_prefix)

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F8 = torch.float8_e4m3fn


class Case:
    """Sequences of `lens` keys (prefix included) over a pool; unowned rows hold `fill`."""

    def __init__(self, lens, prefix, hq=8, hkv=2, d=128, dtype=torch.bfloat16, block=16, kv=None,
                 rel="token", rel_dtype=torch.bfloat16, extent=128, width=None, window=-1,
                 scale=None, seed=0, fill=math.nan):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.prefix, self.block, self.extent, self.window = lens, prefix, block, extent, window
        self.scale = 1.0 / math.sqrt(d) if scale is None else scale
        self.hq, self.hkv, self.d = hq, hkv, d
        n, first = len(lens), prefix // block  # whole blocks of the prefix are the same blocks
        need = [-(-x // block) for x in lens]
        shared = -(-prefix // block)
        pool = shared + sum(max(0, x - first) for x in need) + 3
        order = torch.randperm(pool, generator=g).to(torch.int32).tolist()
        self.prefix_table = torch.tensor(order[:shared], dtype=torch.int32)
        self.table = torch.full((n, max(need + [1])), 1 << 30, dtype=torch.int32)
        self.scales = (0.03, 0.05) if kv == F8 else (1.0, 1.0)
        rows = [torch.randn(prefix, hkv, d, generator=g) for _ in range(2)]
        self.kc, self.vc = (torch.full((pool, block, hkv, d), fill) for _ in range(2))
        for c, x in zip((self.kc, self.vc), rows):
            for j in range(shared):
                part = x[j * block:(j + 1) * block]
                c[order[j], :len(part)] = part
        at = shared
        for b, x in enumerate(lens):
            for j in range(need[b]):
                if j < first:
                    self.table[b, j] = order[j]
                    continue
                blk, at = order[at], at + 1
                self.table[b, j] = blk
                for c, pre in zip((self.kc, self.vc), rows):
                    own = torch.randn(block, hkv, d, generator=g)
                    both = max(0, min(block, prefix - j * block))  # the prefix's last keys, copied
                    own[:both] = pre[j * block:j * block + both]
                    c[blk, :min(block, x - j * block)] = own[:min(block, x - j * block)]
        if kv == F8:
            self.kc, self.vc = ((c / s).to(F8) for c, s in zip((self.kc, self.vc), self.scales))
        else:
            self.kc, self.vc = self.kc.to(dtype), self.vc.to(dtype)
        self.q = torch.randn(n, hq, d, generator=g).to(dtype)
        width = extent if width is None else width
        if rel == "table":
            self.rel = (0.5 * torch.randn(hq, width, generator=g)).to(rel_dtype).expand(n, hq, width)
        else:
            self.rel = (0.5 * torch.randn(n, hq, width, generator=g)).to(rel_dtype)
        self.used = torch.tensor(lens, dtype=torch.int32)
        self.cu = torch.arange(n + 1, dtype=torch.int32)
        self.max_k = max(lens + [0])

    def on(self, dev):
        rel = (self.rel[0].to(dev).expand(self.rel.shape) if self.rel.stride(0) == 0
               else self.rel.to(dev))
        return [x.to(dev) for x in (self.q, self.kc, self.vc)] + [rel] + [
            x.to(dev) for x in (self.cu, self.used, self.table, self.prefix_table)]

    def settings(self):
        return dict(window_size=(self.window, 0) if self.window >= 0 else (-1, -1),
                    softmax_scale=self.scale, return_lse=True, k_scale=self.scales[0],
                    v_scale=self.scales[1])

    def run(self, dev, **kw):
        print(f"shared: {len(self.lens)} sequences {self.lens[:6]} prefix {self.prefix} heads "
              f"{self.hq}/{self.hkv} d {self.d} {self.q.dtype} pool {tuple(self.kc.shape)} "
              f"{self.kc.dtype} extent {self.extent} {self.rel.dtype} window {self.window}", flush=True)
        out, lse = inkling_fa4_rel_attention_decode_shared_prefix(
            *self.on(dev), self.prefix, 1, self.max_k, self.extent, **dict(self.settings(), **kw))
        torch.cuda.synchronize()
        return out.cpu(), lse.cpu()

    def keys(self, b, h):
        """fp64 keys and values of a sequence and kv head; a bad entry's rows are zero."""
        j = torch.arange(self.lens[b])
        ent = self.table[b, j // self.block].long()
        whole = self.prefix // 64 * 64  # read through prefix_table
        ent[:whole] = self.prefix_table[j[:whole] // self.block].long()
        good = (ent >= 0) & (ent < self.kc.shape[0])
        ent = torch.where(good, ent, 0)
        return [torch.where(good[:, None], c[ent, j % self.block, h].double() * s, 0.0)
                for c, s in zip((self.kc, self.vc), self.scales)]

    def check(self, got, rows=None):
        out, lse = got
        h16 = torch.finfo(out.dtype).eps / 2
        for b in range(len(self.lens)) if rows is None else rows:
            lk = self.lens[b]
            lo = max(0, lk - 1 - self.window) if self.window >= 0 else 0
            if lk == 0:
                assert not out[b].any() and lse[:, b].isneginf().all(), b
                continue
            for kv in range(self.hkv):
                heads = slice(kv * (self.hq // self.hkv), (kv + 1) * (self.hq // self.hkv))
                k, v = (x[lo:] for x in self.keys(b, kv))
                q = self.q[b, heads].double()
                x = q @ k.t() * self.scale
                near = min(self.extent, lk - lo)
                if near:
                    x[:, x.shape[1] - near:] += self.rel[b, heads, :near].double().flip(-1)
                want_lse = torch.logsumexp(x, -1)
                live = want_lse > -math.inf
                p = torch.where(live[:, None], torch.softmax(x, -1), 0.0)
                want = p @ v
                big = x.abs().masked_fill(p < 1e-30, 0).amax(-1)  # of the keys that count
                ds = U * ((self.d + 8) * self.scale * (q.abs() @ k.abs().t()).amax(-1) + 8 * big)
                add = (lk + 64) * U
                tol = h16 * want.abs() + (h16 + 2 * ds + add)[:, None] * (p @ v.abs())
                tol += torch.finfo(out.dtype).tiny * torch.finfo(out.dtype).eps
                if out.dtype == torch.float16:
                    tol += 2.0 ** -25 * v.abs().sum(0)
                err = (out[b, heads].double() - want).abs()
                assert (err <= tol).all(), (b, kv, float((err / tol).max()))
                assert (lse[heads, b][~live].isneginf()).all() and not out[b, heads][~live].any()
                err = (lse[heads, b].double() - want_lse)[live].abs()
                tol = (ds + add + 8 * U * want_lse.abs())[live]
                assert (err <= tol).all(), (b, kv, "lse", float((err / tol).max()))


RAGGED = [1000, 1001, 1063, 1064, 1300, 2500, 1017, 1128]


@pytest.mark.parametrize("prefix", [0, 1, 63, 64, 100, 640, 1000])
@pytest.mark.parametrize("block", [8, 16, 64, 256])
def test_prefix_lengths(cuda, prefix, block):
    c = Case(RAGGED, prefix, block=block, seed=prefix + block)
    c.check(c.run(cuda))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (8, 2, 128), (16, 1, 128), (6, 2, 64), (5, 5, 128),
                                      (16, 1, 64), (7, 1, 128)])
def test_heads(cuda, hq, hkv, d, dtype):
    c = Case([900, 832, 833, 1100, 2000], 832, hq, hkv, d, dtype, seed=hq + d)
    c.check(c.run(cuda))


@pytest.mark.parametrize("hq,hkv,d,block", [(8, 2, 128, 16), (4, 4, 64, 16), (16, 1, 128, 8),
                                            (6, 3, 64, 32), (8, 1, 128, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_fp8(cuda, hq, hkv, d, block, dtype):
    c = Case([900, 832, 833, 1100, 2000, 40], 832, hq, hkv, d, dtype, block=block, kv=F8, seed=hq + d)
    c.check(c.run(cuda))


@pytest.mark.parametrize("lens", [[0, 0, 0], [0, 700, 0, 650], [1, 2, 63, 64, 65, 127, 128, 640, 641],
                                  [5], [640], [639, 640, 641], [1, 5000]])
@pytest.mark.parametrize("kv", [None, F8])
def test_sequences_shorter_than_the_prefix_or_empty(cuda, lens, kv):
    c = Case(lens, 640, kv=kv, seed=len(lens))
    c.check(c.run(cuda))


@pytest.mark.parametrize("window", [0, 1, 31, 63, 64, 200, 700, 5000, 2 ** 31 - 1])
@pytest.mark.parametrize("kv", [None, F8])
def test_windows(cuda, window, kv):
    c = Case(RAGGED + [0, 1, 300], 992, window=window, kv=kv, seed=7)
    c.check(c.run(cuda))


@pytest.mark.parametrize("rel", ["token", "table"])
@pytest.mark.parametrize("rel_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("extent,width", [(1, 1), (17, 40), (128, 128), (1024, 1025), (2000, 2000)])
def test_biases(cuda, rel, rel_dtype, extent, width):
    c = Case(RAGGED, 960, rel=rel, rel_dtype=rel_dtype, extent=extent, width=width, seed=extent)
    c.check(c.run(cuda))


def test_no_bias(cuda):
    c = Case(RAGGED, 960, extent=0, width=0, seed=1)
    c.check(c.run(cuda))


@pytest.mark.parametrize("batch", [1, 2, 31, 33, 70, 300])
def test_batches(cuda, batch):
    """Row tiles that a batch fills in part, and more workgroups than fit at once."""
    g = torch.Generator().manual_seed(batch)
    lens = [320 + int(x) for x in torch.randint(0, 90, (batch,), generator=g)]
    c = Case(lens, 320, 6, 2, 64, extent=64, seed=batch)
    c.check(c.run(cuda))


@pytest.mark.parametrize("batch,hq,prefix,own,kv", [
    (256, 8, 4096, 128, None), (200, 8, 4096, 300, None), (200, 8, 4096, 300, F8),
    (80, 4, 9000, 700, None), (24, 16, 2500, 1500, None)])
def test_own_keys_shared_out_over_idle_workgroups(cuda, batch, hq, prefix, own, kv):
    """Workgroups without a prefix piece take several pieces of own keys each, some pieces go to
    the others, and some workgroups of the prefix's range have no piece of it."""
    g = torch.Generator().manual_seed(batch)
    lens = [prefix + int(x) for x in torch.randint(1, own + 1, (batch,), generator=g)]
    lens[3], lens[-1] = prefix + own, 0
    c = Case(lens, prefix, hq, 2, extent=512, kv=kv, seed=batch)
    c.check(c.run(cuda))


@pytest.mark.parametrize("kv", [None, F8])
def test_a_long_prefix_over_small_blocks(cuda, kv):
    """70000 keys in blocks of 16: the window of table entries moves on within a chunk."""
    c = Case([70000 + 5, 70400, 69000], 70000, 2, 1, kv=kv, seed=3)
    c.check(c.run(cuda))


def test_blocks_past_32_bits_of_elements(cuda):
    """The same blocks at the end of a pool of 2^32 elements and more: the same bits."""
    c = Case([700, 650, 1300], 600, block=16, extent=64, seed=18)
    want = c.run(cuda)
    few = c.kc.shape[0]
    shift = (1 << 32) // c.kc[0].numel() + 1000 - few
    pools = []
    for x in (c.kc, c.vc):
        big = torch.empty(shift + few, *x.shape[1:], dtype=x.dtype, device=cuda)
        big[shift:] = x.to(cuda)
        pools.append(big)
    q, _, _, rel, cu, used, table, prefix = c.on(cuda)
    table = torch.where(table < few, table + shift, table)
    out, lse = inkling_fa4_rel_attention_decode_shared_prefix(
        q, *pools, rel, cu, used, table, prefix + shift, c.prefix, 1, c.max_k, c.extent, **c.settings())
    assert torch.equal(out.cpu(), want[0]) and torch.equal(lse.cpu(), want[1])


def test_large_scores(cuda):
    """Scores of +-60 and ramps along the prefix: the running maximum moves many times."""
    c = Case([1500, 1401, 1700], 1400, 4, 2, scale=1.0, rel_dtype=torch.float32, extent=1024, seed=5)
    c.rel = c.rel + torch.linspace(30, -30, 1024)
    c.check(c.run(cuda))


def test_biases_at_the_types_limits(cuda):
    """Lowest finite values and -inf as masks; a row that has nothing else: lowest gives the
    softmax over them, -inf an empty row."""
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        c = Case([700, 650, 641, 30], 640, 4, 2, rel_dtype=dtype, extent=704, seed=6)
        low = torch.finfo(dtype).min
        c.rel[0, 0, 100:300] = low
        c.rel[0, 1, 3:] = -math.inf
        c.rel[1, 0] = -math.inf
        c.rel[1, 1, :] = low
        c.rel[2, 2, :640] = low  # the prefix apart from its first key, and the own key
        c.rel[3, 3, 5:] = low
        got = c.run(cuda)
        assert not got[0][1, 0].any() and got[1][0, 1].isneginf()
        lk = 650
        if dtype != torch.float16:  # all weights alike: the scores vanish next to the bias
            v = c.keys(1, 0)[1]
            mean = v.mean(0)
            tol = 2.0 ** -8 * (mean.abs() + 2 * v.abs().mean(0))
            assert ((got[0][1, 1].double() - mean).abs() <= tol).all()
            assert float(got[1][1, 1]) == pytest.approx(low + math.log(lk), rel=1e-6)
            c.rel[1, 1, :] = 0
            again = c.run(cuda)
            c.check(again)
        else:
            c.check(got)


def test_infinite_keys_outside_a_sequence(cuda):
    """K infinities and NaN in prefix keys that a window hides from all, and in other sequences'
    rows, reach no result."""
    c = Case(RAGGED, 960, window=100, seed=8)
    c.kc[c.prefix_table[0].long()] = math.inf
    c.vc[c.prefix_table[0].long()] = math.nan
    c.check(c.run(cuda))


def test_table_entries_outside_the_pool_read_as_zeros(cuda):
    c = Case([700, 900, 641], 640, seed=9)
    c.prefix_table[3] = c.kc.shape[0]
    c.prefix_table[20] = -1
    c.table[1, 45] = -7
    c.table[0, 41] = 1 << 30
    c.check(c.run(cuda))


def test_lengths_past_the_table_are_clamped(cuda):
    c = Case([640, 704], 640, seed=10)
    c.used = torch.tensor([10 ** 6, -5], dtype=torch.int32)
    out, lse = c.run(cuda)
    c.table[0, 40:44] = c.table[1, 40:44]  # what row 0 names past its end is outside the pool
    assert not out[1].any() and lse[:, 1].isneginf().all()
    assert out[0].isfinite().all()


def test_query_counts_other_than_one(cuda):
    """cu_seqlens_q that is no arange: those sequences' rows are zero, the others right."""
    c = Case([700, 900, 641, 800], 640, seed=11)
    want = c.run(cuda)
    c.cu = torch.tensor([0, 1, 3, 3, 4], dtype=torch.int32)
    out, lse = c.run(cuda)
    assert torch.equal(out[0], want[0][0]) and not out[1:3].any()
    assert lse[:, 1:3].isneginf().all()
    c.cu = torch.tensor([0, 1, 1, 1, 1], dtype=torch.int32)
    out, lse = c.run(cuda)
    assert torch.equal(out[0], want[0][0])


def test_equals_paged_decode(cuda):
    """The same arguments without the prefix: equal up to the rounding of both, twice the bounds
    of one."""
    c = Case([4100, 5000, 4097, 4600], 4096, extent=1024, seed=12)
    a = c.on(cuda)
    got = c.run(cuda)
    out, lse = inkling_fa4_rel_attention_decode_paged(*a[:7], 1, c.max_k, c.extent, bottom_right=True,
                                                      **c.settings())
    c.check(got)
    c.check((out.cpu(), lse.cpu()))


def test_same_bits_every_time_and_without_lse(cuda):
    c = Case([2100, 2500, 2049] * 10, 2048, seed=13)
    first = c.run(cuda)
    for _ in range(2):
        again = c.run(cuda)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    out = inkling_fa4_rel_attention_decode_shared_prefix(
        *c.on(cuda), c.prefix, 1, c.max_k, c.extent, **dict(c.settings(), return_lse=False))
    assert torch.equal(out.cpu(), first[0])


def test_views_and_strides(cuda):
    """q, caches, table and bias as parts of wider tensors."""
    c = Case([700, 900, 641], 640, seed=14)
    want = c.run(cuda)
    q, kc, vc, rel, cu, used, table, pt = c.on(cuda)
    q2 = torch.zeros(3, 12, 128, dtype=q.dtype, device=cuda)
    q2[:, 2:10] = q
    both = torch.stack([kc, vc], 1)
    rel2 = torch.zeros(3, 8, 160, dtype=rel.dtype, device=cuda)
    rel2[..., 1:129] = rel
    table2 = torch.full((3, table.shape[1] + 5), 1 << 30, dtype=torch.int32, device=cuda)
    table2[:, 2:2 + table.shape[1]] = table
    out, lse = inkling_fa4_rel_attention_decode_shared_prefix(
        q2[:, 2:10], both[:, 0], both[:, 1], rel2[..., 1:129], cu, used,
        table2[:, 2:2 + table.shape[1]], pt, c.prefix, 1, c.max_k, c.extent, **c.settings())
    torch.cuda.synchronize()
    assert torch.equal(out.cpu(), want[0]) and torch.equal(lse.cpu(), want[1])


def test_two_streams_at_once(cuda):
    cases = [Case([2100, 2500, 2049] * 4, 2048, seed=s) for s in (15, 16)]
    want = [c.run(cuda) for c in cases]
    args = [c.on(cuda) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(10):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i] = inkling_fa4_rel_attention_decode_shared_prefix(
                    *args[i], c.prefix, 1, c.max_k, c.extent, **c.settings())
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g[0].cpu(), w[0]) and torch.equal(g[1].cpu(), w[1])


def test_graph_replays(cuda):
    """A captured call replayed with other lengths, queries and pages, the program's own work in
    between: the eager result each time."""
    c = Case([2100, 2500, 2049, 2300], 2048, seed=17)
    a = c.on(cuda)

    def step():
        return inkling_fa4_rel_attention_decode_shared_prefix(*a, c.prefix, 1, c.max_k, c.extent,
                                                              **c.settings())
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    for i in range(4):
        a[0].normal_()
        a[5].copy_((c.used - 40 * i).clamp(min=0).to(cuda))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_decode_steps_behind_a_prompt(cuda):
    """A prompt appended once, then steps of four sequences behind it: append, shared decode;
    equal to paged decode over the same cache, and the last step to the definition."""
    prompt, steps, hq, hkv, d, block, n = 200, 5, 8, 2, 128, 16, 4
    g = torch.Generator().manual_seed(18)
    first, own = prompt // block, -(-(prompt + steps) // block) - prompt // block
    pool = first + n * own
    table = torch.zeros(n, first + own, dtype=torch.int32)
    table[:, :first] = torch.arange(first)
    table[:, first:] = torch.arange(first, pool).view(n, own)
    kc, vc = (torch.zeros(pool, block, hkv, d, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    w = (1 + 0.1 * torch.randn(2, d, generator=g)).to(cuda)
    angle = 6.3 * torch.rand(prompt + steps, 32, generator=g).to(cuda)
    on = dict(q_weight=w[0], k_weight=w[1], cos=angle.cos(), sin=angle.sin())
    table = table.to(cuda)

    def tokens(count):
        x = torch.randn(count, hq + 2 * hkv, d, generator=g).to(torch.bfloat16).to(cuda)
        return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    q, k, v = tokens(prompt)
    for b in range(n):  # the prompt's blocks once each; its last part block goes to every sequence
        inkling_fa4_kv_append_paged(k, v, kc, vc, torch.tensor([0, prompt], dtype=torch.int32, device=cuda),
                                    torch.tensor([prompt], dtype=torch.int32, device=cuda),
                                    table[b:b + 1], q=q, **on)
    cu = torch.arange(n + 1, dtype=torch.int32, device=cuda)
    rel = (0.5 * torch.randn(n, hq, 128, generator=g)).to(torch.bfloat16).to(cuda)
    for i in range(steps):
        q, k, v = tokens(n)
        used = torch.full((n,), prompt + i + 1, dtype=torch.int32, device=cuda)
        q = inkling_fa4_kv_append_paged(k, v, kc, vc, cu, used, table, q=q, **on)
        args = (q, kc, vc, rel, cu, used, table)
        out, lse = inkling_fa4_rel_attention_decode_shared_prefix(
            *args, table[0], prompt, 1, prompt + steps, 128, softmax_scale=0.1, return_lse=True)
        ref = inkling_fa4_rel_attention_decode_paged(*args, 1, prompt + steps, 128, softmax_scale=0.1,
                                                     return_lse=True, bottom_right=True)
        torch.cuda.synchronize()
        c = Case.__new__(Case)
        c.lens, c.prefix, c.block, c.extent, c.window, c.scale = [prompt + i + 1] * n, prompt, block, 128, -1, 0.1
        c.hq, c.hkv, c.d, c.scales = hq, hkv, d, (1.0, 1.0)
        c.q, c.kc, c.vc, c.rel, c.table = (x.cpu() for x in (q, kc, vc, rel, table))
        c.prefix_table = c.table[0]
        c.check((out.cpu(), lse.cpu()))
        c.check([x.cpu() for x in ref])


def test_refusals(cuda):
    c = Case([700, 900], 640, seed=19)
    names = ("q", "k_cache", "v_cache", "rel_logits", "cu_seqlens_q", "seqused_k", "block_table",
             "prefix_table")
    ok = dict(zip(names, c.on(cuda)), prefix_len=c.prefix, max_seqlen_q=1, max_seqlen_k=c.max_k,
              rel_extent=c.extent, **c.settings())
    call = inkling_fa4_rel_attention_decode_shared_prefix
    call(**ok)
    kc, pt, q = ok["k_cache"], ok["prefix_table"], ok["q"]
    for bad in (dict(prefix_table=pt[:39]), dict(prefix_table=pt.long()), dict(prefix_table=pt.cpu()),
                dict(prefix_table=pt[None]), dict(prefix_len=-1), dict(prefix_len=pt.numel() * 16 + 1),
                dict(q=q[:1]), dict(q=q.float()), dict(k_cache=kc.half()), dict(k_cache=kc[:, :12]),
                dict(k_cache=kc[:, :12], v_cache=kc[:, :12]),
                dict(max_seqlen_k=ok["block_table"].shape[1] * 16 + 1), dict(rel_extent=129),
                dict(softmax_scale=-1.0), dict(softmax_scale=math.nan),
                dict(k_cache=kc.to(F8), v_cache=kc.to(F8), k_scale=0.0),
                dict(seqused_k=ok["seqused_k"][:1]), dict(block_table=ok["block_table"].long())):
        with pytest.raises(RuntimeError):
            call(**dict(ok, **bad))
    with pytest.raises(ValueError):
        call(**dict(ok, k_cache=kc[0]))
    with pytest.raises(ValueError):
        call(**dict(ok, q=q[:, :7]))


@pytest.mark.parametrize("kv", [None, F8])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 4, 64), (16, 1, 128)])
@pytest.mark.parametrize("window", [0, 5, 40, 130])
def test_own_keys_left_of_the_window_may_hold_anything(cuda, window, hq, hkv, d, kv):
    """NaN and infinite keys and values of a sequence's own that its window hides, the ones next
    to the first visible key among them, reach no result."""
    lens = [640 + n for n in (60, 161, 192, 193, 223, 500, 777)]
    c = Case(lens, 640, hq, hkv, d, kv=kv, window=window, seed=window + d)
    want = c.run(cuda)
    for b, lk in enumerate(lens):
        for j in range(640, lk - 1 - window):
            at = int(c.table[b, j // 16]), j % 16
            c.kc[at] = math.nan
            c.vc[at] = math.nan if j % 2 else (448.0 if kv else math.inf)
    got = c.run(cuda)
    c.check(got)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
