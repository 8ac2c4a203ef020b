"""The fp64 oracle of the head norm and rotation: what a rotation keeps, and its backward
formulas against autograd and central differences (CPU)."""
import pytest
import torch

from oracle.norm_rope import norm_rope, norm_rope_bwd, rotate


def _angles(tokens, rot, seed):
    g = torch.Generator().manual_seed(seed)
    a = 6.0 * torch.rand(tokens, rot // 2, generator=g, dtype=torch.float64)
    return a.cos(), a.sin()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [16, 48, 64])
def test_rotation_keeps_lengths_and_depends_on_the_difference_of_positions(rot, interleaved):
    g = torch.Generator().manual_seed(rot)
    x, y = (torch.randn(1, 3, 64, generator=g, dtype=torch.float64) for _ in range(2))
    theta = torch.rand(rot // 2, generator=g, dtype=torch.float64)

    def turned(v, pos):
        return rotate(v, (pos * theta).cos()[None], (pos * theta).sin()[None], interleaved)
    assert torch.allclose(turned(x, 7).pow(2).sum(-1), x.pow(2).sum(-1), rtol=1e-12)
    a = (turned(x, 11) * turned(y, 4)).sum(-1)
    assert torch.allclose(a, (turned(x, 107) * turned(y, 100)).sum(-1), rtol=1e-10)
    assert torch.equal(turned(x, 5)[..., rot:], x[..., rot:])


def test_half_split_turns_the_first_with_the_one_half_a_rotation_on():
    x = torch.zeros(1, 1, 64, dtype=torch.float64)
    x[..., 2] = 1.0
    cos, sin = _angles(1, 32, 1)
    y = rotate(x, cos, sin)
    assert y[0, 0, 2] == cos[0, 2] and y[0, 0, 18] == sin[0, 2]
    y = rotate(x, cos, sin, interleaved=True)
    assert y[0, 0, 2] == cos[0, 1] and y[0, 0, 3] == sin[0, 1]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [0, 16, 64])
@pytest.mark.parametrize("weight", [False, True])
def test_backward_formulas(rot, interleaved, weight):
    gen = torch.Generator().manual_seed(3)
    f64 = torch.float64
    x = torch.randn(4, 2, 64, generator=gen, dtype=f64, requires_grad=True)
    w = torch.randn(64, generator=gen, dtype=f64, requires_grad=True) if weight else None
    cos, sin = _angles(4, rot, 2) if rot else (None, None)
    g = torch.randn(4, 2, 64, generator=gen, dtype=f64)

    def f(x, w):
        return norm_rope(x, w, cos, sin, 1e-6, interleaved)[0]
    with torch.no_grad():
        dx, dw, _, _ = norm_rope_bwd(x, w, cos, sin, 1e-6, g, interleaved)
        # central differences along a direction: the error is h^2 / 6 times the third
        # derivative, of the order of the values here
        u, h = torch.randn(4, 2, 64, generator=gen, dtype=f64), 1e-5
        diff = ((f(x + h * u, w) - f(x - h * u, w)) * g).sum() / (2 * h)
        assert torch.allclose(diff, (dx * u).sum(), rtol=1e-7, atol=1e-7)
        if weight:
            uw = torch.randn(64, generator=gen, dtype=f64)
            diff = ((f(x, w + h * uw) - f(x, w - h * uw)) * g).sum() / (2 * h)
            assert torch.allclose(diff, (dw * uw).sum(), rtol=1e-7, atol=1e-7)
    want = torch.autograd.grad(f(x, w), [x, w] if weight else [x], g)
    assert torch.allclose(want[0], dx, rtol=1e-10, atol=1e-12)
    if weight:
        assert torch.allclose(want[1], dw, rtol=1e-10, atol=1e-12)
