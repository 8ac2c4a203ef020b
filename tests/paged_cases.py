"""Calls over a paged cache for the tests: sequences whose newest tokens are the queries, the
attention's definition in 64 bits, and bounds on what a kernel may be off by.

Bounds (u = 2^-24; h = half a step of q's type relative to the value; p the weights, n the keys):
  a score is off by at most ds = u ((D + 8) scale sum |q k| + 8 max|s|), the dot product of D
  exact products summed in fp32, its scaling, the bias and the maximum's subtraction; a weight
  by that, exp2's and the rounding to q's type, h; the sums add n u.  So
  out: h |out| + (h + 2 ds + (n + 64) u) A, A = sum p |v| / sum p, and in fp16, where weights
  below 2^-14 of the largest lose bits, 2^-25 sum |v|
  lse: ds + (n + 64) u + 8 u |lse|.
"""
import math

import torch

U = 2.0 ** -24
F8 = torch.float8_e4m3fn


class Case:
    """Sequence b: news[b] queries, lens[b] keys (theirs included) in a pool of blocks; rows that
    no sequence owns hold `fill`, table entries past a sequence's blocks are no blocks.
    layout: "rows" [blocks, block, heads, d]; "heads": heads outermost in a block; "joint": K and
    V side by side in one tensor."""

    def __init__(self, news, lens, hq=8, hkv=2, d=128, dtype=torch.bfloat16, block=16, kv=None,
                 rel="token", rel_dtype=torch.bfloat16, extent=128, width=None, window=-1,
                 causal=True, scale=None, seed=0, fill=math.nan, layout="rows"):
        g = torch.Generator().manual_seed(seed)
        self.news, self.lens, self.block, self.extent = news, lens, block, extent
        self.window, self.causal = window, causal
        self.scale = 1.0 / math.sqrt(d) if scale is None else scale
        self.hq, self.hkv, self.d, self.kv = hq, hkv, d, kv
        n, need = len(lens), [-(-x // block) for x in lens]
        pool = sum(need) + 3
        order = torch.randperm(pool, generator=g).to(torch.int32).tolist()
        self.table = torch.full((n, max(need + [1]) + 1), 1 << 30, dtype=torch.int32)
        self.scales = (0.03, 0.05) if kv == F8 else (1.0, 1.0)
        held = []
        at = 0
        for b, x in enumerate(lens):
            self.table[b, :need[b]] = torch.tensor(order[at:at + need[b]], dtype=torch.int32)
            at += need[b]
        for s in self.scales:
            c = torch.full((pool, block, hkv, d), fill)
            for b, x in enumerate(lens):
                j = torch.arange(x)
                c[self.table[b, j // block].long(), j % block] = torch.randn(x, hkv, d, generator=g)
            held.append((c / s).to(F8) if kv == F8 else c.to(dtype))
        self.kc, self.vc = held
        self.layout = layout
        total = sum(news)
        self.q = torch.randn(total, hq, d, generator=g).to(dtype)
        width = extent if width is None else width
        if rel == "table":
            self.rel = (0.5 * torch.randn(hq, width, generator=g)).to(rel_dtype).expand(total, hq, width)
        else:
            self.rel = (0.5 * torch.randn(total, hq, width, generator=g)).to(rel_dtype)
        self.used = torch.tensor(lens, dtype=torch.int32)
        self.cu = torch.tensor([0] + news, dtype=torch.int32).cumsum(0).to(torch.int32)
        self.max_q, self.max_k = max(news + [0]), max(lens + [0])

    def caches(self, dev):
        k, v = self.kc.to(dev), self.vc.to(dev)
        if self.layout == "heads":
            return [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)]
        if self.layout == "joint":
            both = torch.stack([k.view(torch.uint8), v.view(torch.uint8)], 1).view(k.dtype)
            return [both[:, 0], both[:, 1]]
        return [k, v]

    def on(self, dev):
        rel = (self.rel[0].to(dev).expand(self.rel.shape)
               if self.rel.shape[0] and self.rel.stride(0) == 0 else self.rel.to(dev))
        return [self.q.to(dev)] + self.caches(dev) + [rel] + [
            x.to(dev) for x in (self.cu, self.used, self.table)]

    def settings(self):
        return dict(window_size=(self.window, 0) if self.window >= 0 else (-1, -1),
                    softmax_scale=self.scale, return_lse=True, k_scale=self.scales[0],
                    v_scale=self.scales[1])

    def told(self):
        return (f"news {self.news[:8]} lens {self.lens[:8]} of {len(self.lens)} heads "
                f"{self.hq}/{self.hkv} d {self.d} {self.q.dtype} pool {tuple(self.kc.shape)} "
                f"{self.kc.dtype} extent {self.extent} {self.rel.dtype} window {self.window} "
                f"causal {self.causal} {self.layout}")

    def rows(self, cache, scale, b, h):
        """fp64 rows of a sequence and kv head; a bad entry's rows are zero."""
        j = torch.arange(self.lens[b])
        ent = self.table[b, j // self.block].long()
        good = (ent >= 0) & (ent < cache.shape[0])
        x = cache[torch.where(good, ent, 0), j % self.block, h].double() * scale
        return torch.where(good[:, None], x, 0.0)

    def visible(self, b):
        """[queries, keys] of a sequence."""
        n, lk = self.news[b], self.lens[b]
        dist = (torch.arange(n) + lk - n)[:, None] - torch.arange(lk)
        see = dist >= 0 if self.causal else torch.ones_like(dist, dtype=torch.bool)
        if self.window >= 0:
            see &= dist <= self.window
        return see, dist

    def times(self, b, h):
        """[queries, keys]: how often a query counts a key that the masks leave it (None: once)."""
        return None

    def check(self, got, seqs=None):
        out, lse = got
        h16 = torch.finfo(out.dtype).eps / 2
        group = self.hq // self.hkv
        start = 0
        for b, (n, lk) in enumerate(zip(self.news, self.lens)):
            mine = slice(start, start + n)
            start += n
            if n == 0 or (seqs is not None and b not in seqs):
                continue
            see, dist = self.visible(b)
            for kvh in range(self.hkv):
                k, v = (self.rows(c, s, b, kvh)
                        for c, s in zip((self.kc, self.vc), self.scales))
                times = self.times(b, kvh)
                sees = see if times is None else see & (times > 0)
                for head in range(kvh * group, (kvh + 1) * group):
                    o, ls = out[mine, head].double(), lse[head, mine].double()
                    if lk == 0:
                        assert not o.any() and ls.isneginf().all(), b
                        continue
                    q = self.q[mine, head].double()
                    x = q @ k.t() * self.scale
                    if self.extent:
                        band = (dist >= 0) & (dist < self.extent)
                        rel = self.rel[mine, head].double()
                        x = x + torch.where(
                            band, rel.gather(1, dist.clamp(0, self.extent - 1)), 0.0)
                    if times is not None:
                        x = x + times.double().clamp(min=1).log()
                    x = x.masked_fill(~sees, -math.inf)
                    want_lse = torch.logsumexp(x, -1)
                    live = want_lse > -math.inf
                    p = torch.where(live[:, None], torch.softmax(x, -1), 0.0)
                    want = p @ v
                    big = x.abs().masked_fill(p < 1e-30, 0).amax(-1)  # of the keys that count
                    dots = (q.abs() @ k.abs().t()).masked_fill(~sees, 0).amax(-1)
                    ds = U * ((self.d + 8) * self.scale * dots + 8 * big)
                    add = (lk + 64) * U
                    tol = h16 * want.abs() + (h16 + 2 * ds + add)[:, None] * (p @ v.abs())
                    tol += torch.finfo(out.dtype).tiny * torch.finfo(out.dtype).eps
                    if out.dtype == torch.float16:
                        tol += 2.0 ** -25 * v.abs().sum(0)
                    err = (o - want).abs()
                    assert (err <= tol).all(), (b, head, float((err / tol).max()))
                    assert ls[~live].isneginf().all() and not o[~live].any(), (b, head)
                    err, tol = (ls - want_lse)[live].abs(), (ds + add + 8 * U * want_lse.abs())[live]
                    assert (err <= tol).all(), (b, head, "lse", float((err / tol).max()))
