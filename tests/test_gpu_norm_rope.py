"""Head norm and rotation on the GPU, forward and backward, against the fp64 oracle.

Bounds, elementwise (u = 2^-24, half a step of fp32 relative to the value):
  y   half a step of the output type of |y|, plus 40 u of the terms it is made of: the sum of
      squares rounds at most 13 times (8 in a lane, 4 between lanes, the mean), half of which
      passes to r, its root and quotient 3 times, the products and the sum 6 times
  dx  the same with 80 u: two such sums
  dw  half a step of the weight's type, plus (40 + adds) u of the sum of the terms'
      magnitudes, adds the longest chain of additions: the rows a lane walks over, then the
      lane groups of a workgroup, then the partial rows (in 32 strands)
and one smallest subnormal of the type everywhere.
"""
import math

import pytest
import torch

from inkling_fa4 import inkling_fa4_qk_norm_rope
from oracle.norm_rope import norm_rope, norm_rope_bwd

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-6


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    i = torch.finfo(dtype)
    return i.tiny * i.eps


def _close(got, want, slack, what):
    bound = _half_step(got.dtype) * (want.abs() + slack) + slack + _tiny(got.dtype)
    bad = ~((got.double().cpu() - want).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((got.double().cpu() - want).abs().max()))


def _angles(rows, rot, seed):
    g = torch.Generator().manual_seed(seed)
    a = 6.3 * torch.rand(rows, rot // 2, generator=g)
    return a.cos(), a.sin()


def _inputs(tokens, hq, hkv, d, dtype, wdtype, rot, seed, fused=True):
    g = torch.Generator().manual_seed(seed)
    x = (3 * torch.randn(tokens, hq + 2 * hkv, d, generator=g)).to(dtype)
    w = [(1 + 0.3 * torch.randn(d, generator=g)).to(wdtype) if wdtype else None for _ in range(2)]
    cos, sin = _angles(37, rot, seed) if rot else (None, None)
    pos = torch.randint(0, 37, (tokens,), generator=g).to(torch.int32) if rot else None
    gq, gk = (torch.randn(tokens, h, d, generator=g).to(dtype) for h in (hq, hkv))
    return x[:, :hq], x[:, hq:hq + hkv], w[0], w[1], cos, sin, pos, gq, gk


def _dev(t, dev):
    return None if t is None else t.to(dev)


def _per_token(cos, sin, pos):
    return (None, None) if cos is None else (cos[pos.long()], sin[pos.long()])


def _adds(tokens, heads, d):
    per = 256 // (d // 8)
    blocks = min(-(-tokens // per), 1024)
    return -(-tokens // (blocks * per)) * heads + per + -(-blocks // 32) + 32


def _check(dev, tokens, hq, hkv, d, dtype, wdtype, rot, interleaved, seed=0):
    print(f"norm_rope: tokens {tokens} heads {hq}/{hkv} d {d} {dtype} w {wdtype} rot {rot} "
          f"interleaved {interleaved}", flush=True)
    q, k, qw, kw, cos, sin, pos, gq, gk = _inputs(tokens, hq, hkv, d, dtype, wdtype, rot, seed)
    whole = torch.empty(tokens, hq + 2 * hkv, d, dtype=dtype, device=dev)
    whole[:, :hq], whole[:, hq:hq + hkv] = q.to(dev), k.to(dev)
    leaves = [whole[:, :hq].detach().requires_grad_(), whole[:, hq:hq + hkv].detach().requires_grad_()]
    leaves += [_dev(w, dev).requires_grad_() if w is not None else None for w in (qw, kw)]
    out = inkling_fa4_qk_norm_rope(*leaves, _dev(cos, dev), _dev(sin, dev), _dev(pos, dev), eps=EPS,
                                   interleaved=interleaved)
    named = [x for x in leaves if x is not None]
    grads = list(torch.autograd.grad(out, named, (gq.to(dev), gk.to(dev))))
    if qw is None:
        grads += [None, None]
    torch.cuda.synchronize()
    cs, sn = _per_token(cos, sin, pos)
    for n, (x, w, y, g, dx, dw, heads) in enumerate((
            (q, qw, out[0], gq, grads[0], grads[2], hq), (k, kw, out[1], gk, grads[1], grads[3], hkv))):
        want, size = norm_rope(x, w, cs, sn, EPS, interleaved)
        _close(y, want, 40 * U * size, ("y", n))
        wx, ww, xs, ws = norm_rope_bwd(x, w, cs, sn, EPS, g, interleaved)
        _close(dx, wx, 80 * U * xs, ("dx", n))
        if w is not None:
            _close(dw, ww, (40 + _adds(tokens, heads, d)) * U * ws, ("dw", n))


@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("tokens", [1, 2, 15, 17, 130, 1031])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_lengths(cuda, tokens, d, dtype):
    _check(cuda, tokens, 8, 2, d, dtype, torch.float32, d, False, seed=tokens)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 4), (6, 3), (16, 1), (5, 1), (7, 7)])
def test_heads(cuda, hq, hkv):
    _check(cuda, 65, hq, hkv, 128, torch.bfloat16, torch.bfloat16, 64, True, seed=hq)


@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("rot", [0, 16, 32, 48, 64, 96, 128])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotations(cuda, d, rot, interleaved):
    if rot > d:
        rot = d - 16
    _check(cuda, 77, 6, 2, d, torch.float16, torch.float16, rot, interleaved, seed=rot)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_without_norm(cuda, interleaved):
    _check(cuda, 41, 4, 2, 64, torch.bfloat16, None, 32, interleaved)


def test_more_rows_than_backward_workgroups(cuda):
    _check(cuda, 1024 * 16 + 5, 3, 1, 128, torch.bfloat16, torch.float32, 128, False)


@pytest.mark.parametrize("tokens,hq,hkv,d", [(1, 64, 8, 128), (40, 33, 11, 64), (900, 16, 1, 128),
                                             (5000, 5, 5, 64)])
def test_heads_split_over_workgroups(cuda, tokens, hq, hkv, d):
    """Chunks of heads that hold both kinds, odd counts, and the last chunk short."""
    _check(cuda, tokens, hq, hkv, d, torch.bfloat16, torch.float32, d, False, seed=31)


def test_more_tokens_than_one_launch_takes(cuda):
    """2^25 tokens and some, past 2^31 elements: each row of the outputs is that of its position
    (one input row for all tokens)."""
    tokens, rows = (1 << 25) + 37, 8
    q, k, qw, kw, cos, sin, _, _, _ = _inputs(1, 1, 1, 64, torch.bfloat16, torch.float32, 64, 41)
    x = [t.to(cuda).expand(tokens, 1, 64) for t in (q, k)]
    tables = [_dev(t[:rows], cuda).contiguous() for t in (cos, sin)]
    pos = torch.arange(tokens, device=cuda, dtype=torch.int32) % rows
    out = inkling_fa4_qk_norm_rope(*x, _dev(qw, cuda), _dev(kw, cuda), *tables, pos, eps=EPS)
    few = inkling_fa4_qk_norm_rope(*(t[:rows] for t in x), _dev(qw, cuda), _dev(kw, cuda), *tables,
                                   pos[:rows], eps=EPS)
    for a, b in zip(out, few):
        whole = tokens // rows * rows
        same = (a[:whole].view(-1, rows, 64) == b.view(1, rows, 64)).all(-1).all(0)
        assert same.all() and torch.equal(a[whole:], b[:tokens - whole])


def test_one_weight_only(cuda):
    q, k, qw, kw, cos, sin, pos, _, _ = _inputs(9, 4, 2, 64, torch.bfloat16, torch.float32, 32, 4)
    args = [x.to(cuda) for x in (q, k)], [x.to(cuda) for x in (cos, sin, pos)]
    print("norm_rope: one weight", flush=True)
    a, b = inkling_fa4_qk_norm_rope(*args[0], qw.to(cuda), None, *args[1], eps=EPS)
    cs, sn = _per_token(cos, sin, pos)
    for got, x, w in ((a, q, qw), (b, k, None)):
        want, size = norm_rope(x, w, cs, sn, EPS)
        _close(got, want, 40 * U * size, "one weight")


def test_no_tokens(cuda):
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device=cuda, requires_grad=True)
    w = torch.ones(64, device=cuda, requires_grad=True)
    a, b = inkling_fa4_qk_norm_rope(q, q.detach()[:, :2], w, w.detach())
    assert a.shape == (0, 4, 64) and b.shape == (0, 2, 64)
    gq, gw = torch.autograd.grad(a, (q, w), torch.empty_like(a))
    assert gq.shape == q.shape and torch.equal(gw, torch.zeros_like(w))


def test_gradients_that_are_expanded_sliced_or_missing(cuda):
    """A broadcast gradient (a sum's), one in a wider tensor, an output without one, an input
    that wants none: each equals the contiguous case."""
    q, k, qw, kw, cos, sin, pos, gq, gk = (
        _dev(x, cuda) for x in _inputs(33, 4, 2, 64, torch.float16, torch.float32, 64, 7))
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, qw, kw)]

    def run(inputs, which, g):
        out = inkling_fa4_qk_norm_rope(*leaves, cos, sin, pos)
        return torch.autograd.grad([out[i] for i in which], inputs, g, allow_unused=True)
    ones = torch.ones(1, 1, 1, dtype=torch.float16, device=cuda)
    want = run(leaves, [0, 1], [ones.expand_as(gq).contiguous(), ones.expand_as(gk).contiguous()])
    got = run(leaves, [0, 1], [ones.expand_as(gq), ones.expand_as(gk)])
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    want = run(leaves, [0, 1], [gq, gk])
    wide = torch.zeros(33, 6, 72, dtype=torch.float16, device=cuda)
    wide[:, 1:5, 3:67] = gq  # rows at 6 bytes past a 16-byte boundary
    got = run(leaves, [0, 1], [wide[:, 1:5, 3:67], gk])
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    got = run(leaves, [0], [gq])
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    assert got[1] is None and got[3] is None
    got = run([leaves[3]], [0, 1], [gq, gk])
    assert torch.equal(got[0], want[3])


def test_gradients_that_start_off_a_16_byte_boundary(cuda):
    """Contiguous gradients at an odd offset are as good as aligned ones."""
    x = [_dev(t, cuda) for t in _inputs(9, 3, 2, 64, torch.float16, torch.float32, 64, 21)]
    leaves = [t.clone().requires_grad_() for t in x[:4]]
    want = torch.autograd.grad(inkling_fa4_qk_norm_rope(*leaves, *x[4:7]), leaves, x[7:])

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=cuda)[1:]
        return flat.copy_(t.reshape(-1)).view(t.shape)
    got = torch.autograd.grad(inkling_fa4_qk_norm_rope(*leaves, *x[4:7]), leaves,
                              [shifted(t) for t in x[7:]])
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("absent", [(), (2, 3, 4, 5, 6), (2,), (3,), (4, 5, 6)])
def test_gradients_of_some_inputs(cuda, absent):
    """Each input's gradient asked for by itself, with weights and tables that are not there,
    is the one of the full backward pass."""
    x = [_dev(t, cuda) for t in _inputs(9, 3, 2, 64, torch.bfloat16, torch.float32, 64, 22)]
    x = [None if i in absent else t for i, t in enumerate(x)]
    if all(i in absent for i in (2, 3, 4)):
        x[4:7] = [_dev(t, cuda) for t in _inputs(9, 3, 2, 64, torch.bfloat16, None, 64, 22)[4:7]]
    here = [i for i in range(4) if x[i] is not None]
    for i in here:
        x[i] = x[i].clone().requires_grad_()
    full = torch.autograd.grad(inkling_fa4_qk_norm_rope(*x[:7]), [x[i] for i in here], x[7:])
    for i, want in zip(here, full):
        y = [t if j == i or t is None else t.detach() for j, t in enumerate(x)]
        for leaves in (x, y):  # one leaf of several, and the only one
            out = inkling_fa4_qk_norm_rope(*leaves[:7])
            got, = torch.autograd.grad(out, leaves[i], x[7:])
            assert torch.equal(got, want), i


def test_no_second_derivative(cuda):
    x = [_dev(t, cuda) for t in _inputs(5, 2, 1, 64, torch.bfloat16, torch.float32, 64, 23)]
    leaves = [t.clone().requires_grad_() for t in x[:4]]
    out = inkling_fa4_qk_norm_rope(*leaves, *x[4:7])
    first = torch.autograd.grad(out, leaves, x[7:], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(sum(t.float().sum() for t in first), leaves, allow_unused=True)
    with pytest.raises(ValueError):
        inkling_fa4_qk_norm_rope(*leaves, x[4].clone().requires_grad_(), *x[5:7])


def test_same_bits_every_time(cuda):
    q, k, qw, kw, cos, sin, pos, gq, gk = (
        _dev(x, cuda) for x in _inputs(4099, 8, 2, 128, torch.bfloat16, torch.float32, 128, 9))
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, qw, kw)]
    runs = []
    for _ in range(3):
        out = inkling_fa4_qk_norm_rope(*leaves, cos, sin, pos)
        runs.append(list(out) + list(torch.autograd.grad(out, leaves, (gq, gk))))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


def test_extreme_rows(cuda):
    """Zero rows (only eps under the root), rows at the type's largest values, an infinity or a
    NaN in one row: the others do not change."""
    d, dtype = 64, torch.bfloat16
    q, k, qw, kw, cos, sin, pos, gq, gk = _inputs(8, 4, 2, d, dtype, torch.float32, 16, 11)
    q = q.clone()
    q[0, 0] = 0
    q[1, 1] = 1e18  # its square stays inside fp32
    clean = [_dev(x, cuda) for x in (q, k, qw, kw, cos, sin, pos)]
    a, b = inkling_fa4_qk_norm_rope(*clean, eps=EPS)
    want, size = norm_rope(q, qw, *_per_token(cos, sin, pos), EPS)
    _close(a, want, 40 * U * size, "extreme")
    assert torch.equal(a[0, 0], torch.zeros_like(a[0, 0]))
    bad = clean[0].clone()
    bad[3, 2, 5] = math.inf
    bad[4, 0, 60] = math.nan
    c, e = inkling_fa4_qk_norm_rope(bad, *clean[1:], eps=EPS)
    same = torch.ones(8, 4, dtype=torch.bool, device=cuda)
    same[3, 2] = same[4, 0] = False
    assert torch.equal(a[same], c[same]) and torch.equal(b, e)
    assert c[4, 0].isnan().all()
    # without a norm an element that does not turn passes as it is
    bad = clean[0].clone()
    bad[3, 2, 40] = math.inf
    c, _ = inkling_fa4_qk_norm_rope(bad, clean[1], None, None, *clean[4:])
    assert torch.equal(c[..., 16:], bad[..., 16:])


def test_positions_outside_the_table_stay_inside_it(cuda):
    q, k, qw, kw, cos, sin, pos, _, _ = _inputs(5, 2, 2, 64, torch.bfloat16, torch.float32, 64, 12)
    pos = torch.tensor([-1, -(2 ** 31), 36, 37, 2 ** 31 - 1], dtype=torch.int32)
    a = inkling_fa4_qk_norm_rope(*(_dev(x, cuda) for x in (q, k, qw, kw, cos, sin, pos)))
    near = pos.clamp(0, 36)
    b = inkling_fa4_qk_norm_rope(*(_dev(x, cuda) for x in (q, k, qw, kw, cos, sin, near)))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_tables_with_wider_rows(cuda):
    """cos and sin as column ranges of one table."""
    q, k, qw, kw, cos, sin, pos, _, _ = _inputs(21, 4, 1, 64, torch.bfloat16, torch.float32, 32, 13)
    both = torch.cat([cos, sin], 1).to(cuda)
    x = [_dev(t, cuda) for t in (q, k, qw, kw)]
    a = inkling_fa4_qk_norm_rope(*x, both[:, :16], both[:, 16:], _dev(pos, cuda))
    b = inkling_fa4_qk_norm_rope(*x, _dev(cos, cuda), _dev(sin, cuda), _dev(pos, cuda))
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_other_stream_and_graph(cuda):
    """Forward and backward on a stream of the caller's and in a captured graph, replayed with
    new inputs between the program's own work, equal the eager results."""
    names = _inputs(130, 8, 2, 128, torch.bfloat16, torch.float32, 128, 14)
    q, k, qw, kw, cos, sin, pos, gq, gk = (_dev(x, cuda) for x in names)
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, qw, kw)]

    def step():
        out = inkling_fa4_qk_norm_rope(*leaves, cos, sin, pos)
        return list(out) + list(torch.autograd.grad(out, leaves, (gq, gk)))

    want = [x.detach().clone() for x in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [x.detach() for x in step()]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [x.detach() for x in step()]
    for seed in (15, 16, 17):
        fresh = _inputs(130, 8, 2, 128, torch.bfloat16, torch.float32, 128, seed)
        with torch.no_grad():
            for leaf, x in zip(leaves, fresh):
                leaf.copy_(x.to(cuda))
            gq.copy_(fresh[7].to(cuda))
        graph.replay()
        eager = [x.detach() for x in step()]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, captured))


def test_refusals(cuda):
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=cuda)
    k, w = q[:, :2], torch.ones(64, device=cuda)
    cos = torch.ones(8, 32, device=cuda)
    pos = torch.zeros(3, dtype=torch.int32, device=cuda)
    ok = dict(q=q, k=k, q_weight=w, k_weight=w, cos=cos, sin=cos, positions=pos)
    inkling_fa4_qk_norm_rope(**ok)
    for bad in (dict(q=q.float()), dict(q=q[:2]), dict(q=q.half()), dict(q=q[0]),
                dict(q=q[..., ::2], k=k[..., ::2]), dict(q=q.cpu()), dict(q_weight=w[:32]),
                dict(q_weight=w.bfloat16()), dict(q_weight=w.double(), k_weight=w.double()),
                dict(sin=None), dict(sin=cos[:4]), dict(cos=cos.half(), sin=cos.half()),
                dict(positions=None), dict(positions=pos.long()), dict(positions=pos[:2]),
                dict(positions=pos.cpu()), dict(cos=cos[:, :12], sin=cos[:, :12]),
                dict(cos=cos[:0], sin=cos[:0]), dict(eps=-1.0), dict(eps=math.nan),
                dict(cos=torch.ones(8, 40, device=cuda), sin=torch.ones(8, 40, device=cuda))):
        with pytest.raises(RuntimeError):
            inkling_fa4_qk_norm_rope(**dict(ok, **bad))
    odd = torch.zeros(3 * 4 * 64 + 1, dtype=torch.bfloat16, device=cuda)[1:].view(3, 4, 64)
    with pytest.raises(RuntimeError, match="EUNSUPPORTED"):
        inkling_fa4_qk_norm_rope(**dict(ok, q=odd))


@pytest.mark.parametrize("rms,eps", [(1e13, EPS), (1e14, EPS), (1e16, EPS), (1e18, EPS), (1e-6, 0.0),
                                     (1e-14, 0.0), (1e-16, 0.0), (1e-16, 1e-30)])
def test_backward_of_large_and_small_rows(cuda, rms, eps):
    """Rows whose r^3 leaves fp32 have the gradients of the formula, as the forward its values."""
    d, dtype = 128, torch.bfloat16
    q, k, qw, kw, cos, sin, pos, gq, gk = _inputs(33, 4, 2, d, dtype, torch.float32, 64, 51)
    q, k = ((x.float() * (rms / 3)).to(dtype) for x in (q, k))
    if eps > 0:
        q[2, 1] = 0
    x = [_dev(t, cuda) for t in (q, k, qw, kw, cos, sin, pos, gq, gk)]
    leaves = [t.clone().requires_grad_() for t in x[:4]]
    print(f"norm_rope: rows of rms {rms}, eps {eps}", flush=True)
    out = inkling_fa4_qk_norm_rope(*leaves, *x[4:7], eps=eps)
    grads = torch.autograd.grad(out, leaves, x[7:])
    cs, sn = _per_token(cos, sin, pos)
    eps = float(torch.tensor(eps, dtype=torch.float32))
    for n, (t, w, y, g, heads) in enumerate(((q, qw, out[0], gq, 4), (k, kw, out[1], gk, 2))):
        want, size = norm_rope(t, w, cs, sn, eps)
        _close(y, want, 40 * U * size, ("y", n))
        wx, ww, xs, ws = norm_rope_bwd(t, w, cs, sn, eps, g)
        _close(grads[n], wx, 80 * U * xs, ("dx", n))
        _close(grads[2 + n], ww, (40 + _adds(33, heads, d)) * U * ws, ("dw", n))


def test_strides_of_dimensions_of_one(cuda):
    """The stride of a dimension that holds one row is never stepped along and says nothing."""
    x = _inputs(1, 1, 1, 64, torch.bfloat16, torch.float32, 64, 52)
    q, k, qw, kw, cos, sin, pos, gq, gk = (_dev(t, cuda) for t in x)
    q, k = (t.contiguous().as_strided((1, 1, 64), (64, 64, 1)) for t in (q, k))

    def run(*x):
        leaves = [t.detach().requires_grad_() for t in x] + [w.clone().requires_grad_() for w in (qw, kw)]
        out = inkling_fa4_qk_norm_rope(*leaves, cos, sin, pos)
        return list(out) + list(torch.autograd.grad(out, leaves, (gq, gk)))
    want = run(q, k)
    for st, sh in ((67, 64), (64, 3), (5, 1)):
        got = run(*(t.as_strided((1, 1, 64), (st, sh, 1)) for t in (q, k)))
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    with pytest.raises(RuntimeError, match="EUNSUPPORTED"):  # two rows: stepped along
        inkling_fa4_qk_norm_rope(torch.zeros(134, dtype=torch.bfloat16, device=cuda).as_strided(
            (2, 1, 64), (67, 64, 1)), k.expand(2, 1, 64), qw)


def test_a_table_of_one_row(cuda):
    """cos and sin of one position: the stride between rows says nothing, alike or not."""
    q, k, qw, kw, cos, sin, _, _, _ = (_dev(t, cuda) for t in _inputs(
        5, 2, 1, 64, torch.bfloat16, torch.float32, 32, 53))
    pos = torch.zeros(5, dtype=torch.int32, device=cuda)
    want = inkling_fa4_qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    wide = torch.cat([cos, cos, sin], 1)
    for c in (cos[:1], wide[:1, 16:32], cos[:1].as_strided((1, 16), (3, 1))):
        got = inkling_fa4_qk_norm_rope(q, k, qw, kw, c, sin[:1].clone(), pos)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
