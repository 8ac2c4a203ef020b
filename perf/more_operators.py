"""Long prompts over a paged cache: the operators whose speed is watched, what they are
called with, their plain form, and their values in 64 bits.

  chunk   inkling_fa4_rel_attention_paged: the newest tokens of every sequence attend to
          its paged cache (their own keys included): a chunk of a prompt, draft tokens
  bounds  inkling_fa4_key_bounds_paged: lowest and highest key elements of the blocks that
          new tokens went to
  select  inkling_fa4_select_blocks_paged: for every token and kv head the blocks that its
          attention reads: the first, the last, and the best by the blocks' bounds
  sparse  inkling_fa4_rel_attention_sparse_paged: attention over the blocks so listed

Sizes are this repository's own (Hq 8 / Hkv 2 or Hq = Hkv = 4, head_dim 128 and 64, bias
extents 128 / 512 / 1024, blocks of 16, batches of 8 and of 64 sequences) or odd and ragged
ones of the same ranges.

Fields of a case:
  op, hq, hkv, d, dtype   (of q and the outputs), block, kv ("same" or "fp8")
  batch, q_lo .. q_hi new tokens of a sequence, past_lo .. past_hi keys before them
  rel        chunk, sparse: "token" (a bias row per token and head) or "table" (one per
             head); rel_dtype, extent, window (-1: none), lse
  top, sink, recent   select, sparse: blocks of a list, of them first and last ones
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
_FP8_SCALE = 1.0 / 64  # N(0, 1) keys and values stay inside e4m3's +-448
_BASE = dict(hq=8, hkv=2, d=128, dtype="bf16", block=16, kv="same", batch=1, q_lo=1, q_hi=1,
             past_lo=0, past_hi=0, len_seed=1)
_BIAS = dict(rel="token", rel_dtype="bf16", extent=1024, window=-1, lse=False)
_LIST = dict(top=64, sink=1, recent=2)
_FIELDS = {"chunk": _BIAS, "bounds": {}, "select": _LIST, "sparse": {**_BIAS, **_LIST}}


def _case(op, **kw):
    return dict(_BASE, op=op, **dict(_FIELDS[op], **kw))


def listed():
    return [
        # Draft tokens of a few sequences of the small model to be verified: latency counts.
        _case("chunk", name="chunk_verify_8x4", batch=8, q_lo=4, q_hi=4, past_lo=100,
              past_hi=2000, hq=4, hkv=4, d=64, dtype="fp16", rel="table", rel_dtype="fp32",
              extent=128),
        # One chunk of a long prompt, a global layer.
        _case("chunk", name="chunk_512_16k", q_lo=512, q_hi=512, past_lo=15872, past_hi=15872),
        # A mixed serving step on an fp8 cache: chunks of prompts beside short turns.
        _case("chunk", name="chunk_ragged_fp8", batch=16, q_lo=3, q_hi=500, past_lo=90,
              past_hi=8000, kv="fp8", lse=True),
        # A local layer of the same kind of step.
        _case("chunk", name="chunk_window_24", batch=24, q_lo=1, q_hi=300, past_lo=300,
              past_hi=4000, hq=6, hkv=2, block=32, extent=512, window=511),
        # A full batch of long conversations, each with a long new turn: matrix products.
        _case("chunk", name="chunk_8x2048", batch=8, q_lo=2048, q_hi=2048, past_lo=6144,
              past_hi=6144, rel="table", rel_dtype="fp32", extent=128),
        # After the append of a decode step.
        _case("bounds", name="bounds_step_64", batch=64, past_lo=1000, past_hi=32000),
        # After the append of a batch of long prompts.
        _case("bounds", name="bounds_prompts_8x4096", batch=8, q_lo=4096, q_hi=4096),
        # A decode step over long caches.
        _case("select", name="select_step_64", batch=64, past_lo=2000, past_hi=32700, top=128),
        # A chunk of a long prompt, on an fp8 cache.
        _case("select", name="select_chunk_fp8", q_lo=512, q_hi=512, past_lo=30000, past_hi=30000,
              kv="fp8", top=100),
        # A few sequences, larger blocks: latency counts.
        _case("sparse", name="sparse_step_4", batch=4, past_lo=5000, past_hi=20000, hq=4, hkv=4,
              d=64, dtype="fp16", rel="table", rel_dtype="fp32", extent=128, block=64, top=16),
        # The attention of a decode step over long caches.
        _case("sparse", name="sparse_step_64", batch=64, past_lo=2000, past_hi=32700, top=128),
        # The attention of a chunk of a long prompt, on an fp8 cache, with the LSE.
        _case("sparse", name="sparse_chunk_fp8", q_lo=512, q_hi=512, past_lo=30000, past_hi=30000,
              kv="fp8", top=100, lse=True),
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
    op = rng.choice(["chunk", "chunk", "chunk", "bounds", "select", "select", "sparse", "sparse"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    c = dict(hq=hq, hkv=hkv, d=rng.choice([128, 128, 128, 64]), dtype=dtype,
             block=rng.choice([16, 16, 32, 64]), kv=rng.choice(["same", "same", "fp8"]),
             len_seed=rng.randrange(1 << 20))
    if op != "chunk" and rng.random() < 0.5:  # a decode step
        c["batch"] = _log_int(rng, 1, 128)
    else:
        c["batch"] = _log_int(rng, 1, 32)
        c["q_lo"], c["q_hi"] = _span(rng, 2, 4096 if op == "bounds" else 2048)
    c["past_lo"], c["past_hi"] = _span(rng, 1, 32768)
    if op in ("chunk", "sparse"):
        c["extent"] = rng.choice([128, 512, 1024])
        c["rel"] = rng.choice(["token", "token", "table"])
        c["rel_dtype"] = rng.choice([dtype, "fp32"])
        c["lse"] = rng.random() < 0.3
        c["window"] = c["extent"] - 1 if op == "chunk" and rng.random() < 0.25 else -1
    if op in ("select", "sparse"):
        c["top"] = max(4, _log_int(rng, 256, 4096) // c["block"])
        c["sink"], c["recent"] = rng.randint(0, 2), rng.randint(1, 2)
        least = 2 * c["top"] * c["block"]  # there is a choice to make
        c["past_lo"], c["past_hi"] = max(c["past_lo"], least), max(c["past_hi"], 2 * least)
    return _case(op, **c)


def _plain_bytes(c):
    """About what the plain form holds at once."""
    lens = _lens(c)
    most_q, most_k = max(n for n, _ in lens), max(n + past for n, past in lens)
    tokens, blocks = sum(n for n, _ in lens), most_k // c["block"] + 1
    if c["op"] == "chunk":
        return 4 * c["batch"] * most_k * (c["hq"] * most_q + 2 * c["hkv"] * c["d"])
    if c["op"] == "bounds":
        return 4 * c["batch"] * most_q * c["hkv"] * c["d"]
    if c["op"] == "select":
        return 8 * c["batch"] * blocks * c["hkv"] * (2 * c["d"] + 2 * most_q)
    return 8 * tokens * c["hkv"] * c["top"] * c["block"] * c["d"]


def draw(rng):
    most = [work(c) for c in listed()]
    flops, nbytes = max(w["flops"] for w in most), max(w["bytes"] for w in most)
    plain = max(_plain_bytes(c) for c in listed())
    while True:
        c = _draw(rng)
        w = work(c)
        if w["flops"] / flops + w["bytes"] / nbytes <= 1.0 and _plain_bytes(c) <= plain:
            return c


def _lens(c):
    """New tokens of each sequence, and the keys before them."""
    r = random.Random(c["len_seed"])
    return [(r.randint(c["q_lo"], c["q_hi"]), r.randint(c["past_lo"], c["past_hi"]))
            for _ in range(c["batch"])]


def _esize(name):
    return {"fp8": 1, "fp32": 4}.get(name, 2)


def _sum_min(lo, hi, most):
    """Sum of min(x, most) over lo <= x < hi."""
    cut = min(max(most, lo), hi)
    return (lo + cut - 1) * (cut - lo) // 2 + (hi - cut) * most


def work(case):
    """Inputs and outputs once: keys that some query sees, the bias that a visible key needs,
    table entries and lengths.  Attention 4 d flops per visible pair and head, scores 4 d per
    block, token and kv head, bounds two comparisons an element."""
    c = case
    lens, bs, d = _lens(c), c["block"], c["d"]
    tokens, kv = sum(n for n, _ in lens), _esize(c["kv"] if c["kv"] == "fp8" else c["dtype"])
    nbytes = 4 * (2 * c["batch"] + 1)
    pairs = band = keys = blocks = 0
    for n, past in lens:
        lk = n + past
        if c["op"] == "chunk":
            most = c["window"] + 1 if c["window"] >= 0 else lk
            pairs += _sum_min(past + 1, lk + 1, most)
            band += _sum_min(past + 1, lk + 1, min(most, c["extent"]))
            seen = min(lk, most + n - 1)
            keys, blocks = keys + seen, blocks + -(-seen // bs)
        elif c["op"] == "bounds":
            first = past // bs * bs
            keys, blocks = keys + lk - first, blocks + -(-lk // bs) - past // bs
        elif c["op"] == "select":
            blocks += -(-lk // bs)
            pairs += sum(p // bs + 1 for p in range(past, lk))  # blocks a token chooses from
        else:
            rows = [(min(p + 1, (c["top"] - 1) * bs + p % bs + 1), p) for p in range(past, lk)]
            pairs += sum(r for r, _ in rows)
            band += sum(min(r, c["extent"], p + 1, c["recent"] * bs) for r, p in rows)
            listed_keys = min(lk, sum(r for r, _ in rows))
            keys, blocks = keys + listed_keys, blocks + -(-listed_keys // bs)
    nbytes += 4 * blocks
    if c["op"] == "bounds":
        nbytes += c["hkv"] * d * kv * (keys + 2 * blocks)
        return {"bytes": nbytes, "flops": 2 * c["hkv"] * d * keys}
    if c["op"] == "select":
        nbytes += tokens * (2 * c["hq"] * d + 4 * c["hkv"] * c["top"])
        nbytes += 2 * blocks * c["hkv"] * d * kv
        return {"bytes": nbytes, "flops": 4 * d * pairs * c["hkv"]}
    nbytes += 2 * tokens * c["hq"] * d * 2 + 2 * keys * c["hkv"] * d * kv
    nbytes += c["hq"] * _esize(c["rel_dtype"]) * (band if c["rel"] == "token" else c["extent"])
    nbytes += 4 * tokens * c["hq"] if c["lse"] else 0
    if c["op"] == "sparse":
        nbytes += 4 * tokens * c["hkv"] * c["top"]
    return {"bytes": nbytes, "flops": 4 * d * pairs * c["hq"]}


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages(lens, block, g):
    """Block table of sequences of `lens` keys, and the blocks of the pool."""
    counts = [-(-n // block) for n in lens]
    order = torch.randperm(sum(counts), generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(counts), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(counts)


def _positions(s, tokens):
    """Sequence and position of each token."""
    n = s["cu_q"][1:] - s["cu_q"][:-1]
    seq = torch.repeat_interleave(torch.arange(n.numel(), device="cuda"), n.long(),
                                  output_size=tokens)
    return seq, (s["used"] - s["cu_q"][1:])[seq].long() + torch.arange(tokens, device="cuda")


def _choose(score, pos, c):
    """The lists of tokens at positions pos from scores [tokens, hkv, blocks], which this
    changes: first and last blocks, the best of the rest, lower blocks first where equal."""
    blk = torch.arange(score.shape[2], device="cuda")
    last = (pos // c["block"])[:, None, None]
    score[score.isnan()] = math.inf
    fixed = (blk < c["sink"]) | (blk > last - c["recent"])
    rank = fixed.to(score.dtype)  # 1: always, 0: by the score, -1: never
    rank = torch.where(blk > last, -1.0, rank).expand(score.shape)
    score = torch.sort(score, dim=-1, descending=True, stable=True)
    order = torch.sort(rank.gather(2, score.indices), dim=-1, descending=True, stable=True)
    best = score.indices.gather(2, order.indices)[..., :c["top"]]
    best = torch.where(order.values[..., :c["top"]] < 0, 1 << 30, best)
    if best.shape[2] < c["top"]:
        best = torch.nn.functional.pad(best, (0, c["top"] - best.shape[2]), value=1 << 30)
    best = best.sort(-1).values
    return torch.where(best == 1 << 30, -1, best).to(torch.int32)


def prepare(case, seed):
    c = case
    g = torch.Generator("cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    lens, dtype = _lens(c), _DTYPES[c["dtype"]]
    hq, hkv, d, bs = c["hq"], c["hkv"], c["d"], c["block"]
    keys, tokens = [n + past for n, past in lens], sum(n for n, _ in lens)
    s = {"case": c, "max_q": max(n for n, _ in lens), "max_k": max(keys)}
    s["table"], blocks = _pages(keys, bs, g)
    s["used"], s["cu_q"] = _int32(keys), _int32([0] + [n for n, _ in lens]).cumsum(0).int()

    def held(x):
        return (x / _FP8_SCALE).to(torch.float8_e4m3fn) if c["kv"] == "fp8" else x.to(dtype)

    if c["op"] in ("bounds", "select"):
        # of 16 keys of N(0, 1) and more, lowest and highest lie around -1.8 and 1.8
        far = 0.5 * randn(blocks, hkv, 2, d) + _int32([-2, 2])[:, None]
        s["bounds"] = held(far.sort(2).values)
    if c["op"] != "select":
        s["k_cache"] = held(randn(blocks, bs, hkv, d))
    if c["op"] == "bounds":
        return s
    s["q"] = randn(tokens, hq, d).to(dtype)
    if c["op"] == "select":
        return s
    s["v_cache"] = held(randn(blocks, bs, hkv, d))
    rdtype = _DTYPES[c["rel_dtype"]]
    if c["rel"] == "table":
        s["rel"] = (0.5 * randn(hq, c["extent"])).to(rdtype).expand(tokens, hq, c["extent"])
    else:
        s["rel"] = (0.5 * randn(tokens, hq, c["extent"])).to(rdtype)
    if c["op"] == "sparse":
        # the tokens of a sequence rate its blocks alike, but not the same
        seq, pos = _positions(s, tokens)
        most = s["table"].shape[1]
        score = randn(c["batch"], hkv, most)[seq]
        score += 0.7 * randn(tokens, hkv, most)
        s["blocks"] = _choose(score, pos, c)
    return s


# ---- plain forms ---------------------------------------------------------------------------


def _scales(c):
    return _FP8_SCALE if c["kv"] == "fp8" else 1.0


def _bias(c, rel, dist):
    """Bias rows [..., extent] at distances dist [..., keys], zero off the band."""
    off = (dist < 0) | (dist >= c["extent"])
    return rel.gather(-1, dist.clamp(0, c["extent"] - 1)).masked_fill_(off, 0.0)


def _softmax(x, v):
    """Softmax of x [..., rows, keys] times v [..., keys, d], and the log of its sum."""
    m = x.amax(-1, keepdim=True)
    w = (x - m).exp_()
    total = w.sum(-1, keepdim=True)
    return (w @ v) / total, (m + total.log())[..., 0]


def _plain_chunk(s, c):
    batch, hq, hkv, d, bs = c["batch"], c["hq"], c["hkv"], c["d"], c["block"]
    group, tokens, nq = hq // hkv, s["q"].shape[0], s["max_q"]
    first = s["cu_q"][:-1].long()
    n = (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    # queries and bias rows of a sequence side by side, the short ones filled with their last
    row = first[:, None] + torch.minimum(torch.arange(nq, device="cuda"), n[:, None] - 1)
    q = s["q"][row].float().view(batch, nq, hkv, group, d).permute(0, 2, 3, 1, 4) / d
    nk = s["table"].shape[1] * bs
    k, v = (s[name][s["table"].long()].view(batch, nk, hkv, d).transpose(1, 2).float() * _scales(c)
            for name in ("k_cache", "v_cache"))
    x = (q.reshape(batch, hkv, group * nq, d) @ k.transpose(2, 3)).view(batch, hq, nq, nk)
    pos = (s["used"].long() - n)[:, None] + row - first[:, None]
    dist = pos[:, :, None] - torch.arange(nk, device="cuda")
    x += _bias(c, s["rel"][row].float().transpose(1, 2), dist[:, None].expand(x.shape))
    hidden = dist < 0
    if c["window"] >= 0:
        hidden |= dist > c["window"]
    x.masked_fill_(hidden[:, None], -math.inf)
    o, lse = _softmax(x.view(batch, hkv, group * nq, nk), v)
    seq, pos = _positions(s, tokens)
    at = pos - (s["used"].long() - n)[seq]
    out = {"out": o.view(batch, hq, nq, d)[seq, :, at].to(s["q"].dtype)}
    if c["lse"]:
        out["lse"] = lse.view(batch, hq, nq)[seq, :, at].t().contiguous()
    return out


def _plain_bounds(s, c):
    bs = c["block"]
    used, n = s["used"].long(), (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    first, last = (used - n) // bs, (used - 1) // bs
    # the blocks of a sequence that changed, the short lists filled with its last block
    most = (s["max_q"] + bs - 2) // bs + 1
    blk = torch.minimum(first[:, None] + torch.arange(most, device="cuda"), last[:, None])
    at = s["table"].gather(1, blk).long()
    keys = s["k_cache"][at].float()  # [batch, most, block, hkv, d]
    row = blk[:, :, None] * bs + torch.arange(bs, device="cuda")
    gone = (row >= used[:, None, None])[..., None, None]
    lo = keys.masked_fill(gone, math.inf).amin(2)
    hi = keys.masked_fill(gone, -math.inf).amax(2)
    new = torch.stack([lo, hi], -2).to(s["bounds"].dtype)
    held = torch.uint8 if c["kv"] == "fp8" else s["bounds"].dtype  # bytes: indexing moves them
    s["bounds"].view(held)[at] = new.view(held)
    return {"bounds": s["bounds"]}


def _plain_select(s, c):
    # in 64 bits: 32 decide blocks of nearly equal scores by the order of a sum
    batch, hkv, d, tokens, nq = c["batch"], c["hkv"], c["d"], s["q"].shape[0], s["max_q"]
    first = s["cu_q"][:-1].long()
    n = (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    row = first[:, None] + torch.minimum(torch.arange(nq, device="cuda"), n[:, None] - 1)
    q = s["q"].double().view(tokens, hkv, c["hq"] // hkv, d)
    q = torch.stack([q.clamp(max=0.0).sum(2), q.clamp(min=0.0).sum(2)], 2)  # as lowest, highest
    b = s["bounds"][s["table"].long()].double().flatten(3).permute(0, 2, 3, 1)
    score = q.flatten(2)[row].transpose(1, 2) @ b  # [batch, hkv, nq, blocks]
    seq, pos = _positions(s, tokens)
    at = pos - (s["used"].long() - n)[seq]
    return {"blocks": _choose(score[seq, :, at], pos, c)}


def _plain_sparse(s, c):
    hq, hkv, d, bs, tokens = c["hq"], c["hkv"], c["d"], c["block"], s["q"].shape[0]
    seq, pos = _positions(s, tokens)
    blk = s["blocks"].long()
    at = s["table"][seq[:, None, None], blk.clamp(min=0)].long()
    head = torch.arange(hkv, device="cuda")[:, None]
    k, v = (s[name].transpose(1, 2)[at, head].view(tokens, hkv, -1, d).float() * _scales(c)
            for name in ("k_cache", "v_cache"))
    key = (blk[..., None] * bs + torch.arange(bs, device="cuda")).view(tokens, hkv, 1, -1)
    dist = pos[:, None, None, None] - key
    q = s["q"].float().view(tokens, hkv, hq // hkv, d) / d
    x = q @ k.transpose(2, 3)
    x += _bias(c, s["rel"].float().view(tokens, hkv, hq // hkv, -1), dist.expand(x.shape))
    hidden = (dist < 0) | (key < 0)
    if c["window"] >= 0:
        hidden |= dist > c["window"]
    x.masked_fill_(hidden, -math.inf)
    o, lse = _softmax(x, v)
    out = {"out": o.view(tokens, hq, d).to(s["q"].dtype)}
    if c["lse"]:
        out["lse"] = lse.view(tokens, hq).t().contiguous()
    return out


# ---- one pass ------------------------------------------------------------------------------


def _framework():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import inkling_fa4
    return inkling_fa4


def _attention_options(c):
    kw = dict(k_scale=_FP8_SCALE, v_scale=_FP8_SCALE) if c["kv"] == "fp8" else {}
    return dict(kw, window_size=(c["window"], 0) if c["window"] >= 0 else (-1, -1),
                return_lse=c["lse"])


def _attention_outputs(c, out):
    return {"out": out[0], "lse": out[1]} if c["lse"] else {"out": out}


def _own_chunk(s, c):
    return _attention_outputs(c, _framework().inkling_fa4_rel_attention_paged(
        s["q"], s["k_cache"], s["v_cache"], s["rel"], s["cu_q"], s["used"], s["table"], s["max_q"],
        s["max_k"], c["extent"], **_attention_options(c)))


def _own_bounds(s, c):
    _framework().inkling_fa4_key_bounds_paged(s["k_cache"], s["bounds"], s["cu_q"], s["used"],
                                              s["table"], s["max_q"])
    return {"bounds": s["bounds"]}


def _own_select(s, c):
    return {"blocks": _framework().inkling_fa4_select_blocks_paged(
        s["q"], s["bounds"], s["cu_q"], s["used"], s["table"], c["block"], s["max_q"], s["max_k"],
        c["top"], sink_blocks=c["sink"], recent_blocks=c["recent"])}


def _own_sparse(s, c):
    return _attention_outputs(c, _framework().inkling_fa4_rel_attention_sparse_paged(
        s["q"], s["k_cache"], s["v_cache"], s["rel"], s["cu_q"], s["used"], s["table"],
        s["blocks"], s["max_q"], s["max_k"], c["extent"], **_attention_options(c)))


_PLAIN = {"chunk": _plain_chunk, "bounds": _plain_bounds, "select": _plain_select,
          "sparse": _plain_sparse}
_OWN = {"chunk": _own_chunk, "bounds": _own_bounds, "select": _own_select, "sparse": _own_sparse}


def run(state):
    c = state["case"]
    if own:
        return _OWN[c["op"]](state, c)
    with torch.no_grad():
        return _PLAIN[c["op"]](state, c)


# ---- values in 64 bits ---------------------------------------------------------------------


def _rows(s, name, b, lk, h, bs):
    """Keys or values 0 .. lk - 1 of sequence b and kv head h, in 64 bits."""
    at = s["table"][b, :-(-lk // bs)].long()
    x = s[name][:, :, h][at]
    return x.reshape(-1, x.shape[-1])[:lk].double()


def _attend(q, k, v, bias, hidden):
    x = (q @ k.t() + bias).masked_fill(hidden, -math.inf)
    return torch.softmax(x, -1) @ v, torch.logsumexp(x, -1)


def _exact_bias(c, rel, dist):
    """Bias of one head, rows [queries, extent], at dist [queries, keys]."""
    wide = torch.cat([rel.double(), torch.zeros(rel.shape[0], 1, dtype=torch.float64,
                                                device=rel.device)], 1)
    none = torch.full_like(dist, c["extent"])
    return wide.gather(1, torch.where((dist >= 0) & (dist < c["extent"]), dist, none))


def _exact_attention(c, s):
    bs, group, tokens = c["block"], c["hq"] // c["hkv"], s["q"].shape[0]
    out = torch.zeros(tokens, c["hq"], c["d"], dtype=torch.float64, device="cuda")
    lse = torch.zeros(c["hq"], tokens, dtype=torch.float64, device="cuda")
    start = 0
    for b, (n, past) in enumerate(_lens(c)):
        lk = n + past
        for h in range(c["hkv"]):
            k, v = (_rows(s, name, b, lk, h, bs) * _scales(c) for name in ("k_cache", "v_cache"))
            for i0 in range(0, n, 512):
                i1 = min(n, i0 + 512)
                dist = (torch.arange(past + i0, past + i1, device="cuda")[:, None]
                        - torch.arange(lk, device="cuda"))
                hidden = dist < 0
                if c["window"] >= 0:
                    hidden = hidden | (dist > c["window"])
                mine = slice(start + i0, start + i1)
                if c["op"] == "sparse":
                    named = torch.zeros(i1 - i0, -(-lk // bs) + 1, device="cuda")
                    named.scatter_(1, (s["blocks"][mine, h].long() % named.shape[1]), 1.0)
                    named = named[:, :-1].repeat_interleave(bs, 1)[:, :lk]  # -1: the last column
                    hidden = hidden | (named == 0)
                for head in range(h * group, (h + 1) * group):
                    bias = _exact_bias(c, s["rel"][mine, head], dist)
                    out[mine, head], lse[head, mine] = _attend(
                        s["q"][mine, head].double() / c["d"], k, v, bias, hidden)
        start += n
    return {"out": out, "lse": lse} if c["lse"] else {"out": out}


def _exact_bounds(c, s):
    bs, bounds = c["block"], s["bounds"].double()
    for b, (n, past) in enumerate(_lens(c)):
        lk = n + past
        for h in range(c["hkv"]):
            k = _rows(s, "k_cache", b, lk, h, bs)[past // bs * bs:]
            pad = -k.shape[0] % bs
            if pad:
                k = torch.cat([k, k[-1:].expand(pad, -1)])
            k = k.view(-1, bs, c["d"])
            at = s["table"][b, past // bs:-(-lk // bs)].long()
            bounds[at, h, 0], bounds[at, h, 1] = k.min(1).values, k.max(1).values
    return {"bounds": bounds}


def _exact_select(c, s):
    group, start, lists = c["hq"] // c["hkv"], 0, []
    for b, (n, past) in enumerate(_lens(c)):
        bound = s["bounds"][s["table"][b, :-(-(n + past) // c["block"])].long()].double()
        for i0 in range(0, n, 8):
            q = s["q"][start + i0:start + min(n, i0 + 8)].double()
            pos = torch.arange(past + i0, past + i0 + q.shape[0], device="cuda")
            score = torch.stack([sum(
                torch.maximum(q[:, h * group + e, None] * bound[None, :, h, 0],
                              q[:, h * group + e, None] * bound[None, :, h, 1]).sum(-1)
                for e in range(group)) for h in range(c["hkv"])], 1)
            lists.append(_choose(score, pos, c))
        start += n
    return {"blocks": torch.cat(lists)}


def exact(case, seed):
    c = case
    if c["op"] == "select" and work(c)["flops"] > 2e10:
        return None
    s = prepare(c, seed)
    if c["op"] == "bounds":
        return _exact_bounds(c, s)
    return _exact_select(c, s) if c["op"] == "select" else _exact_attention(c, s)
