"""The operators around paged attention whose speed is watched: what they are
called with, their plain form, and their values in 64 bits.

  norm    inkling_fa4_qk_norm_rope: RMS norm of every query and key head, then the
          rotation by the token's position; forward, or forward and backward
  append  inkling_fa4_kv_append_paged: the same norm and rotation of new tokens, keys
          and values written to a paged cache (16 bits or e4m3), queries returned
  shared  inkling_fa4_rel_attention_decode_shared_prefix: one query per sequence over a
          paged cache whose first prefix_len keys are the same blocks for all sequences

Sizes are this repository's own (Hq 8 / Hkv 2 or Hq = Hkv = 4, head_dim 128 and 64,
bias extents 128 / 512 / 1024, blocks of 16, batches of 8 x 4096 tokens and of 64 decoded
sequences) or odd and ragged ones of the same ranges.

Fields of a case:
  op, hq, hkv, d, dtype   (of q, k, v and the outputs)
  rope       "none", "half" (element i turns with i + rot / 2) or "pairs" (2 i with 2 i + 1)
  rot        leading elements of a head that turn; wdtype: type of the norm weights
  norm       tokens, seqs (positions count from 0 in each), train
  append     batch, q_lo .. q_hi new tokens of a sequence, past_lo .. past_hi keys before
             them, block, kv ("same" or "fp8"), normed (k and q are normed)
  shared     batch, prefix, own_lo .. own_hi keys after the prefix, block, kv, rel ("token": a
             bias row per sequence and head, "table": one per head), rel_dtype, extent,
             window (-1: none), lse
  len_seed   of the lengths
"""
import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.getcwd(), "inkling-fa4-relative-attention_amd")
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-6
_FP8_SCALE = 1.0 / 64  # N(0, 1) keys and values stay inside e4m3's +-448
_BASE = dict(op="norm", hq=8, hkv=2, d=128, dtype="bf16", rope="half", rot=128, wdtype="bf16",
             len_seed=1)


def _norm(**kw):
    return dict(_BASE, **dict(dict(tokens=512, seqs=1, train=False), **kw))


def _append(**kw):
    return dict(_BASE, **dict(dict(op="append", batch=1, q_lo=1, q_hi=1, past_lo=0, past_hi=0,
                                   block=16, kv="same", normed=True), **kw))


def _shared(**kw):
    c = dict(_BASE, **dict(dict(op="shared", batch=64, prefix=4096, own_lo=1, own_hi=512, block=16,
                                kv="same", rel="token", rel_dtype="bf16", extent=1024, window=-1,
                                lse=False), **kw))
    for unused in ("rope", "rot", "wdtype"):
        del c[unused]
    return c


def listed():
    return [
        # A short prompt of the small model on its way to the prefill.
        _norm(name="norm_prompt_512", tokens=512, hq=4, hkv=4, d=64, rot=64, dtype="fp16",
              wdtype="fp32"),
        # A training step over the throughput workload's batch, forward and backward.
        _norm(name="norm_train_8x4096", tokens=8 * 4096, seqs=8, train=True),
        # A ragged training batch: three query heads to a kv head, half of a head turns, in
        # neighbouring pairs.
        _norm(name="norm_train_ragged", tokens=4987, seqs=7, train=True, hq=6, hkv=2, d=64, rot=32,
              rope="pairs", dtype="fp16", wdtype="fp32"),
        # A serving decode step: one token of each of 64 sequences.
        _append(name="append_step_64", batch=64, past_lo=16, past_hi=2048),
        # Chunked prefill on an fp8 cache, positions by the relative bias alone (no rotation).
        _append(name="append_chunk_fp8", batch=16, q_lo=100, q_hi=128, past_lo=0, past_hi=256,
                rope="none", rot=0, kv="fp8"),
        # A full batch of long prompts going into the cache.
        _append(name="append_prompts_8x4096", batch=8, q_lo=4096, q_hi=4096, wdtype="fp32"),
        # A few sequences of the small model behind a short prompt: latency counts.
        _shared(name="shared_4x512", batch=4, prefix=512, own_hi=64, hq=4, hkv=4, d=64,
                dtype="fp16", rel="table", rel_dtype="fp32", extent=128),
        # A serving decode step of a global layer, 64 sequences behind one long document.
        _shared(name="shared_64x16k", prefix=16384, own_hi=1024),
        # The same on an fp8 cache with more sequences, and the LSE a caller merges by.
        _shared(name="shared_128x8k_fp8", batch=128, prefix=8192, kv="fp8", lse=True),
        # A local layer: the window passes the prefix's end for some sequences only.
        _shared(name="shared_window_48", batch=48, prefix=4080, own_hi=700, hq=16, hkv=2,
                window=511, extent=512),
        # Many samples of one very long prompt: bound by the matrix products.
        _shared(name="shared_256x32k", batch=256, prefix=32768, own_hi=256),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _span(rng, lo, hi):
    """Two sizes lo <= a <= b <= hi, spread over the logarithm."""
    a, b = sorted((_log_int(rng, lo, hi), _log_int(rng, lo, hi)))
    return a, b


_HEADS = ((4, 4), (8, 2), (8, 2), (8, 4), (16, 4), (8, 1), (6, 3), (16, 2), (6, 2))


def _draw(rng):
    hq, hkv = rng.choice(_HEADS)
    d = rng.choice([128, 128, 128, 64])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    rope = rng.choice(["half", "half", "pairs", "none"])
    c = dict(hq=hq, hkv=hkv, d=d, dtype=dtype, rope=rope,
             rot=0 if rope == "none" else rng.choice([d, d, d // 2, 16]),
             wdtype=rng.choice([dtype, "fp32"]), len_seed=rng.randrange(1 << 20))
    op = rng.choice(["norm", "norm", "append", "append", "shared", "shared", "shared"])
    if op == "norm":
        tokens = _log_int(rng, 1, 32768)
        return _norm(**dict(c, tokens=tokens, seqs=rng.randint(1, min(8, tokens)),
                            train=rng.random() < 0.6))
    kv, block = rng.choice(["same", "same", "fp8"]), rng.choice([16, 16, 32, 64])
    if op == "append":
        normed = rope == "none" or rng.random() < 0.8
        if rng.random() < 0.5:
            lens = dict(batch=_log_int(rng, 1, 256))
            lens["past_lo"], lens["past_hi"] = _span(rng, 1, 2048)
        else:
            lens = dict(batch=_log_int(rng, 1, 16))
            lens["q_lo"], lens["q_hi"] = _span(rng, 2, 2048)
            lens["past_lo"], lens["past_hi"] = _span(rng, 1, 1024)
        return _append(**dict(c, kv=kv, block=block, normed=normed, **lens))
    lo, hi = _span(rng, 1, 2048)
    extent = rng.choice([128, 512, 1024])
    prefix = block * max(1, _log_int(rng, 256, 32768) // block)
    del c["rope"], c["rot"], c["wdtype"]
    return _shared(**dict(c, batch=_log_int(rng, 2, 256), prefix=prefix, own_lo=lo, own_hi=hi, kv=kv,
                          block=block, rel=rng.choice(["token", "token", "table"]),
                          rel_dtype=rng.choice([dtype, "fp32"]), extent=extent,
                          window=extent - 1 if rng.random() < 0.25 else -1,
                          lse=rng.random() < 0.3))


def draw(rng):
    most = [work(c) for c in listed()]
    flops, nbytes = max(w["flops"] for w in most), max(w["bytes"] for w in most)
    while True:
        c = _draw(rng)
        w = work(c)
        if w["flops"] / flops + w["bytes"] / nbytes <= 1.0 and _dense_keys(c) <= 9_000_000:
            return c


def _dense_keys(c):
    """Query-key pairs of a shared case, the prefix of all and the longest own part."""
    return c["batch"] * (c["prefix"] + c["own_hi"]) if c["op"] == "shared" else 0


def _lens(c):
    """Lengths of each sequence: norm: tokens; append: (new, before); shared: own keys."""
    r = random.Random(c["len_seed"])
    if c["op"] == "norm":
        cuts = sorted(r.sample(range(1, c["tokens"]), c["seqs"] - 1))
        return [b - a for a, b in zip([0] + cuts, cuts + [c["tokens"]])]
    if c["op"] == "append":
        return [(r.randint(c["q_lo"], c["q_hi"]), r.randint(c["past_lo"], c["past_hi"]))
                for _ in range(c["batch"])]
    return [r.randint(c["own_lo"], c["own_hi"]) for _ in range(c["batch"])]


def _esize(name):
    return 4 if name == "fp32" else 2


def work(case):
    """Inputs and outputs once: rows of the turn's table that some token needs, pages and
    lengths; attention: every key that some sequence sees once, the bias that a visible key
    needs, 4 d flops per visible pair and head.  Norm and turn: 8 flops an element."""
    c = case
    lens = _lens(c)
    if c["op"] == "shared":
        pairs = band = 0
        first, last = c["prefix"], 0  # keys of the prefix that some sequence sees
        keys = 0
        for n in lens:
            lk = c["prefix"] + n
            lo = max(0, lk - 1 - c["window"]) if c["window"] >= 0 else 0
            pairs += lk - lo
            band += lk - max(lo, lk - c["extent"])
            if lo < c["prefix"]:
                first, last = min(first, lo), c["prefix"]
            keys += lk - max(lo, c["prefix"])
        keys += max(0, last - first)
        nbytes = 2 * c["batch"] * c["hq"] * c["d"] * 2
        nbytes += 2 * keys * c["hkv"] * c["d"] * (1 if c["kv"] == "fp8" else 2)
        nbytes += c["hq"] * _esize(c["rel_dtype"]) * (band if c["rel"] == "token" else c["extent"])
        nbytes += 4 * keys // c["block"] + (4 * c["batch"] * c["hq"] if c["lse"] else 0)
        return {"bytes": nbytes, "flops": 4 * c["d"] * pairs * c["hq"]}
    if c["op"] == "norm":
        tokens, rows, held = c["tokens"], max(lens), 0
        passes = 5 if c["train"] else 2
        nbytes = passes * tokens * (c["hq"] + c["hkv"]) * c["d"] * 2
        flops = 8 * tokens * (c["hq"] + c["hkv"]) * c["d"] * (3 if c["train"] else 1)
    else:
        tokens = sum(n for n, _ in lens)
        rows = len({p for n, past in lens for p in range(past, past + n)})
        held = 1 if c["kv"] == "fp8" else 2
        nbytes = tokens * c["d"] * (4 * c["hq"] + 2 * c["hkv"] * (2 + held)) + 8 * len(lens)
        nbytes += 4 * sum(-(-(n + past) // c["block"]) - past // c["block"] for n, past in lens)
        flops = 8 * tokens * (c["hq"] + c["hkv"]) * c["d"]
    if c["rope"] != "none":
        nbytes += 4 * rows * c["rot"] + (4 * tokens if c["op"] == "norm" else 0)
    nbytes += 2 * c["d"] * _esize(c["wdtype"])
    return {"bytes": nbytes, "flops": flops}


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return _int32(out)


def _pages(lens, block, g, first=0):
    """Block table of sequences of `lens` keys and the blocks of the pool; the first `first`
    columns name the same blocks in every row."""
    counts = [-(-n // block) for n in lens]
    total = first + sum(n - first for n in counts)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(counts), dtype=torch.int32, device="cuda")
    table[:, :first] = order[:first]
    at = first
    for b, n in enumerate(counts):
        table[b, first:n] = order[at:at + n - first]
        at += n - first
    return table, total


def _turn_table(c, rows):
    """cos, sin [rows, rot / 2] of the usual angles, from 64 bits."""
    i = torch.arange(c["rot"] // 2, dtype=torch.float64, device="cuda")
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
        -2.0 * i / c["rot"])
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    c = case
    g = torch.Generator("cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    lens, dtype = _lens(c), _DTYPES[c["dtype"]]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    s = {"case": c}
    if c["op"] == "shared":
        block, first = c["block"], c["prefix"] // c["block"]
        keys = [c["prefix"] + n for n in lens]
        s["table"], blocks = _pages(keys, block, g, first)
        s["prefix_table"] = s["table"][0, :first].clone()
        s["used"], s["cu_q"], s["max_k"] = _int32(keys), _cu([1] * len(lens)), max(keys)
        s["q"] = randn(c["batch"], hq, d).to(dtype)
        for name in ("k_cache", "v_cache"):
            x = randn(blocks, block, hkv, d)
            s[name] = (x / _FP8_SCALE).to(torch.float8_e4m3fn) if c["kv"] == "fp8" else x.to(dtype)
        rdtype = _DTYPES[c["rel_dtype"]]
        if c["rel"] == "table":
            s["rel"] = (0.5 * randn(hq, c["extent"])).to(rdtype).expand(c["batch"], hq, c["extent"])
        else:
            s["rel"] = (0.5 * randn(c["batch"], hq, c["extent"])).to(rdtype)
        return s
    if c["op"] == "norm":
        tokens, rows = c["tokens"], max(lens)
        s["positions"] = torch.cat([torch.arange(n, dtype=torch.int32, device="cuda") for n in lens])
    else:
        tokens, keys = sum(n for n, _ in lens), [n + past for n, past in lens]
        rows = max(keys)
        s["cu_q"], s["used"] = _cu([n for n, _ in lens]), _int32(keys)
        s["table"], blocks = _pages(keys, c["block"], g)
        held = torch.float8_e4m3fn if c["kv"] == "fp8" else dtype
        for name in ("k_cache", "v_cache"):
            s[name] = randn(blocks, c["block"], hkv, d).to(held)
    # q, k and v are column ranges of one projection's output
    qkv = randn(tokens, hq + 2 * hkv, d).to(dtype)
    s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    s["qw"], s["kw"] = ((1 + 0.1 * randn(d)).to(_DTYPES[c["wdtype"]]) for _ in range(2))
    if c["op"] == "append" and not c["normed"]:
        s["qw"] = s["kw"] = None
    s["cos"], s["sin"] = _turn_table(c, rows) if c["rope"] != "none" else (None, None)
    if c["op"] == "norm" and c["rope"] == "none":
        s["positions"] = None
    if c["op"] == "norm" and c["train"]:
        s["gq"], s["gk"] = randn(tokens, hq, d).to(dtype), randn(tokens, hkv, d).to(dtype)
        for name in ("q", "k", "qw", "kw"):
            s[name] = s[name].detach().requires_grad_()
    return s


# ---- plain forms ---------------------------------------------------------------------------


def _normed(x, w):
    x = x.float()
    if w is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w.float()


def _turned(c, x, cos, sin, back=False):
    """x [tokens, heads, d] turned by cos, sin [tokens, rot / 2]; back: the other way round."""
    if c["rope"] == "none":
        return x
    cos, sin = cos[:, None], -sin[:, None] if back else sin[:, None]
    turn, rest = x[..., :c["rot"]], x[..., c["rot"]:]
    if c["rope"] == "half":
        a, b = turn[..., :c["rot"] // 2], turn[..., c["rot"] // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = turn[..., 0::2], turn[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _norm_back(x, w, g):
    """Gradients of x and w of the norm, from that of its output."""
    x = x.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    xh, gw = x * r, g * w.float()
    return r * (gw - xh * (gw * xh).mean(-1, keepdim=True)), (g * xh).sum((0, 1))


def _plain_norm(s, c):
    rows = s["positions"].long() if s["positions"] is not None else None
    cos, sin = (s["cos"][rows], s["sin"][rows]) if rows is not None else (None, None)
    out = {}
    for n in ("q", "k"):
        out[n] = _turned(c, _normed(s[n], s[n + "w"]), cos, sin).to(s[n].dtype)
    if c["train"]:
        for n in ("q", "k"):
            gx, gw = _norm_back(s[n], s[n + "w"], _turned(c, s["g" + n].float(), cos, sin, True))
            out["d" + n], out["d" + n + "w"] = gx.to(s[n].dtype), gw.to(s[n + "w"].dtype)
    return out


def _slots(s, c):
    """Position of each new token, its block and its row in it."""
    n = s["cu_q"][1:] - s["cu_q"][:-1]
    seq = torch.repeat_interleave(torch.arange(c["batch"], device="cuda"), n.long(),
                                  output_size=s["k"].shape[0])
    pos = (s["used"] - s["cu_q"][1:])[seq].long() + torch.arange(s["k"].shape[0], device="cuda")
    return pos, s["table"][seq, pos // c["block"]].long(), pos % c["block"]


def _plain_append(s, c):
    pos, blk, row = _slots(s, c)
    cos, sin = (s["cos"][pos], s["sin"][pos]) if s["cos"] is not None else (None, None)
    k, v = _turned(c, _normed(s["k"], s["kw"]), cos, sin), s["v"].float()
    q = _turned(c, _normed(s["q"], s["qw"]), cos, sin).to(s["q"].dtype)
    if c["kv"] == "fp8":
        k, v = ((x / _FP8_SCALE).clamp(-448.0, 448.0) for x in (k, v))
    for cache, x in ((s["k_cache"], k), (s["v_cache"], v)):
        cache.view(torch.uint8)[blk, row] = x.to(cache.dtype).view(torch.uint8)
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_shared(s, c):
    bs, hkv, d, batch, p = c["block"], c["hkv"], c["d"], c["batch"], c["prefix"]
    group, mul = c["hq"] // hkv, _FP8_SCALE if c["kv"] == "fp8" else 1.0
    q = s["q"].float().view(batch, hkv, group, d) / d
    qp = q.transpose(0, 1).reshape(hkv, batch * group, d)
    kp, vp = (s[n][s["prefix_table"].long()].reshape(p, hkv, d).transpose(0, 1).float() * mul
              for n in ("k_cache", "v_cache"))  # [hkv, p, d]
    mine = s["table"][:, p // bs:].long()
    n_own = mine.shape[1] * bs
    ko, vo = (s[n][mine].reshape(batch, n_own, hkv, d).transpose(1, 2).float() * mul
              for n in ("k_cache", "v_cache"))  # [batch, hkv, n_own, d]
    x = torch.cat([(qp @ kp.transpose(1, 2)).view(hkv, batch, group, p).transpose(0, 1),
                   q @ ko.transpose(2, 3)], -1).view(batch, c["hq"], p + n_own)
    key = torch.arange(p + n_own, device="cuda")
    dist = (s["used"] - 1)[:, None] - key
    bias = s["rel"].float().gather(2, dist.clamp(0, c["extent"] - 1)[:, None].long().expand(
        batch, c["hq"], p + n_own))
    x += bias.masked_fill_(((dist < 0) | (dist >= c["extent"]))[:, None], 0.0)
    hidden = dist < 0
    if c["window"] >= 0:
        hidden |= dist > c["window"]
    x.masked_fill_(hidden[:, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    w = (x - m).exp_()
    total = w.sum(-1, keepdim=True)
    wp = w[..., :p].view(batch, hkv, group, p).transpose(0, 1).reshape(hkv, batch * group, p)
    o = (wp @ vp).view(hkv, batch, group, d).transpose(0, 1)
    o = (o + w[..., p:].reshape(batch, hkv, group, n_own) @ vo).reshape(batch, c["hq"], d)
    out = {"out": (o / total).to(s["q"].dtype)}
    if c["lse"]:
        out["lse"] = (m + total.log())[..., 0].t().contiguous()
    return out


# ---- one pass ------------------------------------------------------------------------------


def _framework():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import inkling_fa4
    return inkling_fa4


def _own_norm(s, c):
    q, k = _framework().inkling_fa4_qk_norm_rope(
        s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], s["positions"], eps=_EPS,
        interleaved=c["rope"] == "pairs")
    if not c["train"]:
        return {"q": q, "k": k}
    names = ("q", "k", "qw", "kw")
    grads = torch.autograd.grad((q, k), [s[n] for n in names], (s["gq"], s["gk"]))
    return {"q": q, "k": k, **{"d" + n: x for n, x in zip(names, grads)}}


def _own_append(s, c):
    kw = dict(k_scale=_FP8_SCALE, v_scale=_FP8_SCALE) if c["kv"] == "fp8" else {}
    q = _framework().inkling_fa4_kv_append_paged(
        s["k"], s["v"], s["k_cache"], s["v_cache"], s["cu_q"], s["used"], s["table"], q=s["q"],
        q_weight=s["qw"], k_weight=s["kw"], cos=s["cos"], sin=s["sin"], eps=_EPS,
        interleaved=c["rope"] == "pairs", **kw)
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_shared(s, c):
    kw = dict(k_scale=_FP8_SCALE, v_scale=_FP8_SCALE) if c["kv"] == "fp8" else {}
    out = _framework().inkling_fa4_rel_attention_decode_shared_prefix(
        s["q"], s["k_cache"], s["v_cache"], s["rel"], s["cu_q"], s["used"], s["table"],
        s["prefix_table"], c["prefix"], 1, s["max_k"], c["extent"],
        window_size=(c["window"], 0) if c["window"] >= 0 else (-1, -1), return_lse=c["lse"], **kw)
    return {"out": out[0], "lse": out[1]} if c["lse"] else {"out": out}


_PLAIN = {"norm": _plain_norm, "append": _plain_append, "shared": _plain_shared}
_OWN = {"norm": _own_norm, "append": _own_append, "shared": _own_shared}


def run(state):
    c = state["case"]
    if own:
        return _OWN[c["op"]](state, c)
    with torch.no_grad():
        return _PLAIN[c["op"]](state, c)


# ---- values in 64 bits ---------------------------------------------------------------------


def _turn_matrices(c, cos, sin):
    """The turn of a token as a matrix [tokens, d, d]: y = x @ M."""
    d, half = c["d"], c["rot"] // 2
    m = torch.eye(d, dtype=torch.float64, device="cuda").repeat(cos.shape[0], 1, 1)
    i = torch.arange(half, device="cuda")
    a, b = (i, i + half) if c["rope"] == "half" else (2 * i, 2 * i + 1)
    m[:, a, a], m[:, b, b], m[:, a, b], m[:, b, a] = cos, cos, sin, -sin
    return m


def _exact_rows(c, x, w, cos, sin, g=None):
    """Norm and turn of x [tokens, heads, d] in 64 bits, blocks of tokens; with g, the output's
    gradient: those of x and w too (by autograd)."""
    w = w.detach().double().requires_grad_() if w is not None else None
    outs, grads = [], []
    dw = torch.zeros_like(w) if w is not None else None
    for at in range(0, x.shape[0], 4096):
        xb = x[at:at + 4096].detach().double().requires_grad_()
        y = xb
        if w is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / c["d"] + _EPS).sqrt() * w
        if cos is not None:
            y = y @ _turn_matrices(c, cos[at:at + 4096].double(), sin[at:at + 4096].double())
        if g is not None:
            gx, gw = torch.autograd.grad(y, (xb, w), g[at:at + 4096].double())
            grads.append(gx)
            dw += gw
        outs.append(y.detach())
    return torch.cat(outs), torch.cat(grads) if grads else None, dw


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] == "norm":
        rows = s["positions"].long() if s["positions"] is not None else None
        cos, sin = (s["cos"][rows], s["sin"][rows]) if rows is not None else (None, None)
        out = {}
        for n in ("q", "k"):
            y, gx, gw = _exact_rows(c, s[n], s[n + "w"], cos, sin, s.get("g" + n))
            out[n] = y
            if c["train"]:
                out["d" + n], out["d" + n + "w"] = gx, gw
        return out
    if c["op"] == "append":
        pos = torch.cat([torch.arange(past, past + n, device="cuda") for n, past in _lens(c)])
        cos, sin = (s["cos"][pos], s["sin"][pos]) if s["cos"] is not None else (None, None)
        rows = {"k": _exact_rows(c, s["k"], s["kw"], cos, sin)[0], "v": s["v"].double()}
        out = {"q": _exact_rows(c, s["q"], s["qw"], cos, sin)[0]}
        for n in ("k", "v"):
            cache, x = s[n + "_cache"].double(), rows[n]
            if c["kv"] == "fp8":
                x = (x / _FP8_SCALE).clamp(-448, 448).to(torch.float8_e4m3fn).double()
            at = 0
            for b, (new, past) in enumerate(_lens(c)):
                p = torch.arange(past, past + new, device="cuda")
                cache[s["table"][b].long()[p // c["block"]], p % c["block"]] = x[at:at + new]
                at += new
            out[n + "_cache"] = cache
        return out
    mul = _FP8_SCALE if c["kv"] == "fp8" else 1.0
    out = torch.zeros(c["batch"], c["hq"], c["d"], dtype=torch.float64, device="cuda")
    lse = torch.zeros(c["hq"], c["batch"], dtype=torch.float64, device="cuda")
    group = c["hq"] // c["hkv"]
    for b, lk in enumerate(s["used"].tolist()):
        lo = max(0, lk - 1 - c["window"]) if c["window"] >= 0 else 0
        at = s["table"][b, lo // c["block"]:-(-lk // c["block"])].long()
        skip = lo // c["block"] * c["block"]
        near = min(c["extent"], lk - lo)  # the last keys carry bias
        for h in range(c["hkv"]):
            k, v = (s[n][at][:, :, h].reshape(-1, c["d"])[lo - skip:lk - skip].double() * mul
                    for n in ("k_cache", "v_cache"))
            heads = slice(h * group, (h + 1) * group)
            x = s["q"][b, heads].double() @ k.t() / c["d"]
            x[:, -near:] += s["rel"][b, heads, :near].double().flip(-1)
            out[b, heads] = torch.softmax(x, -1) @ v
            lse[heads, b] = torch.logsumexp(x, -1)
    return {"out": out, "lse": lse} if c["lse"] else {"out": out}
