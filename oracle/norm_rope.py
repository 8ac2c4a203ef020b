"""RMS norm of head rows, the position rotation, and the paged append (test oracle).

The reference has none of these as code; its serving caller norms q and k per head
before the attention and writes a paged cache (outputs/architecture.md:24-50,117-127).
Semantics restated, in fp64:
  z = x (mean(x^2) + eps)^-1/2 w    (w None: z = x)
  the pair (a, b) of the rot leading elements -> (a cos - b sin, b cos + a sin), pairs
  (i, i + rot / 2) or, interleaved, (2 i, 2 i + 1), angles of the token's position
  backward: rotation by the negative angles, then
  dx = r w g - x r^3 / D sum(w g x),  dw = sum over rows of g x r

TEST INFRASTRUCTURE: imported only by tests.
Pinned by tests/test_oracle_norm_rope.py: norms and inner products under the rotation,
the backward formulas against autograd and central differences.
"""
import torch


def _pairs(rot, interleaved):
    i = torch.arange(rot // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)


def rotate(x, cos, sin, interleaved=False):
    """x [tokens, heads, D] turned by cos, sin [tokens, rot / 2]; fp64."""
    y = x.double().clone()
    if cos is None:
        return y
    ia, ib = _pairs(2 * cos.shape[1], interleaved)
    c, s = cos.double()[:, None], sin.double()[:, None]
    a, b = x.double()[..., ia], x.double()[..., ib]
    y[..., ia] = a * c - b * s
    y[..., ib] = b * c + a * s
    return y


def norm_rope(x, w, cos, sin, eps, interleaved=False):
    """(y, size of the terms that make it up) in fp64; cos, sin per token or None."""
    z = x.double()
    if w is not None:
        z = z * (z.pow(2).mean(-1, keepdim=True) + eps).rsqrt() * w.double()
    y = rotate(z, cos, sin, interleaved)
    size = z.abs()
    if cos is not None:
        ia, ib = _pairs(2 * cos.shape[1], interleaved)
        size = size.clone()
        size[..., ia] = size[..., ib] = z[..., ia].abs() + z[..., ib].abs()
    return y, size


def norm_rope_bwd(x, w, cos, sin, eps, g, interleaved=False):
    """(dx, dw, size of dx's terms, size of dw's terms) in fp64; dw None without w."""
    gz = rotate(g, cos, None if sin is None else -sin, interleaved)
    gsize = norm_rope(g, None, cos, None if sin is None else -sin, eps, interleaved)[1]
    if w is None:
        return gz, None, gsize, None
    x, w = x.double(), w.double()
    d = x.shape[-1]
    r = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    f = r ** 3 / d
    dx = r * gz * w - x * f * (gz * w * x).sum(-1, keepdim=True)
    dw = (gz * x * r).sum((0, 1))
    dx_size = r * gsize * w.abs() + x.abs() * f * (gsize * (w * x).abs()).sum(-1, keepdim=True)
    return dx, dw, dx_size, (gsize * x.abs() * r).sum((0, 1))


def append_positions(cu_seqlens, seqused_k):
    """(sequence, position) of every new token that belongs to a sequence."""
    cu = cu_seqlens.tolist()
    for b, used in enumerate(seqused_k.tolist()):
        for t in range(cu[b], cu[b + 1]):
            yield t, b, used - (cu[b + 1] - t)
