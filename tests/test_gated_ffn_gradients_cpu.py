"""The gradients that the feed-forward block is held to, against central differences of its definition, both in 64 bits: what stands
behind the element-wise bounds of the kernel's tests does not rest on the formulas that the kernel was written from.

A central difference with step h along a unit direction is off by h^2 / 6 of the third derivative and by 2^-52 / h of the sum of the
terms' magnitudes; at h = 1e-4 and these sizes (terms of some 10^4, derivatives of the order of the slope) both are below 1e-6 of
a slope along the gradient, which is its length."""
import pytest
import torch
from test_gated_ffn_gpu import reference

SIZES = [(1, 16, 8), (5, 24, 40), (70, 136, 264)]


def inputs(t, c, f):
    g = torch.Generator().manual_seed(1000 * t + c + f)
    n = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)
    return [n(t, c), n(2 * f, c) * 0.7 * c ** -0.5, n(c, f) * 0.7 * f ** -0.5], n(t, c)


def slope_along(base, dy, k, d, h=1e-4):
    """Of sum(dy * y) along d in operand k."""
    def y(x, wgu, wd):
        f = wd.shape[1]
        gate, up = x @ wgu[:f].T, x @ wgu[f:].T
        return (gate / (1 + torch.exp(-gate)) * up) @ wd.T
    plus, minus = list(base), list(base)
    plus[k], minus[k] = base[k] + h * d, base[k] - h * d
    return float(((y(*plus) - y(*minus)) * dy).sum() / (2 * h))


@pytest.mark.parametrize("t,c,f", SIZES)
def test_the_formulas(t, c, f):
    base, dy = inputs(t, c, f)
    grads, _ = reference(*base, dy=dy)
    gen = torch.Generator().manual_seed(1)
    for k, g in enumerate(grads):
        length = float(g.norm())
        along = g / g.norm()
        across = torch.randn(g.shape, generator=gen, dtype=torch.float64)
        across /= across.norm()
        agrees = lambda grad, d: abs(float((grad * d).sum()) - slope_along(base, dy, k, d)) <= 1e-6 * length
        assert agrees(g, along) and agrees(g, across), k
        # a gradient that is missing, turned round or a thousandth off is seen
        for wrong in (torch.zeros_like(g), -g, 1.001 * g):
            assert not agrees(wrong, along), k


@pytest.mark.parametrize("half", ["gate", "up"])
def test_that_a_wrong_half_is_seen(half):
    """The two halves of dw_gate_up are checked each by itself: one of them zero does not hide behind the other."""
    base, dy = inputs(70, 136, 264)
    g = reference(*base, dy=dy)[0][1]
    rows = slice(0, 264) if half == "gate" else slice(264, 528)
    d = torch.zeros_like(g)
    d[rows] = g[rows] / g[rows].norm()
    slope = slope_along(base, dy, 1, d)
    assert abs(float((g * d).sum()) - slope) <= 1e-6 * float(g.norm())
    without = g.clone()
    without[rows] = 0
    assert abs(float((without * d).sum()) - slope) > 0.1 * float(g.norm())
