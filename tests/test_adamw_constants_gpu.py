"""AdamW with a coefficient forms its constants in 64 bits, without one in fp32 from rounded betas. Both against 64 bits at the usual
betas, and against each other at a coefficient of one.

fp32 rounds a beta in [1/2, 1) by at most 2^-25; 1 - beta is then exact, so it is off by at most D = 2^-25. beta^t is off by at most
t D, and 2^-23 for the power, and 2^-24 for the difference from one. Everything else is at most eight fp32 operations a moment and
sixteen more to the update, of 2^-24 each, of the values and of what the constants are off by."""
import math

import pytest
import torch

from sirius_b200 import ops

pytestmark = pytest.mark.gpu
U, D = 2.0 ** -24, 2.0 ** -25
LR, EPS, WD = 3e-4, 1e-8, 0.01


def state(n):
    g = torch.Generator(device="cuda").manual_seed(n)
    r = lambda s: torch.randn(n, device="cuda", generator=g) * s
    return [r(0.05), r(1e-2), r(1e-3), r(1e-2).square()]   # p, g, m, v


def step64(p, g, m, v, b1, b2, t):
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    scale = LR / (1 - b1 ** t) / (v1.sqrt() / math.sqrt(1 - b2 ** t) + EPS)
    return p * (1 - LR * WD) - scale * m1, m1, v1, scale


def bounds(p, g, m, v, b1, b2, t, rounded):
    """Of p, m and v: the fp32 operations, and with `rounded` betas what the constants are off by."""
    _, m1, v1, scale = step64(p, g, m, v, b1, b2, t)
    up = scale * m1.abs()
    d = D if rounded else 0.0
    off = (t * D + 3 * U) if rounded else 0.0
    em = 8 * U * (b1 * m.abs() + (1 - b1) * g.abs()) + d * (m.abs() + g.abs())
    ev = 10 * U * v1 + d * (v + g * g)
    # half of v's and of its correction's relative errors, all of the other correction's
    ep = 4 * U * p.abs() + 32 * U * up + em * scale + up * (0.51 * (ev / v1) + 1.01 * off / (1 - b1 ** t) + 0.51 * off / (1 - b2 ** t))
    return ep, em, ev


@pytest.mark.parametrize("b1,b2", [(0.9, 0.999), (0.9, 0.95), (0.8, 0.9999), (0.875, 0.9375)])
@pytest.mark.parametrize("t", [1, 7, 1000])
def test_both_ways_to_form_the_constants(b1, b2, t):
    n = 4099
    with_clip, without = state(n), state(n)
    clip = ops.grad_norm([with_clip[1]], 1e6)
    assert float(clip[1]) == 1.0
    p, g, m, v = (x.double() for x in state(n))
    ops.adamw(*with_clip, LR, b1, b2, EPS, WD, t, clip=clip)
    ops.adamw(*without, LR, b1, b2, EPS, WD, t)
    want = step64(p, g, m, v, b1, b2, t)
    for got, rounded, what in ((with_clip, False, "with"), (without, True, "without")):
        bound = bounds(p, g, m, v, b1, b2, t, rounded)
        for k, x, e in ((0, want[0], bound[0]), (2, want[1], bound[1]), (3, want[2], bound[2])):
            worst = ((got[k].double() - x).abs() - e).max()
            assert worst <= 0, (what, "pgmv"[k], float(worst))
    # of each other: the difference is that of the constants
    exact = b1 == 0.875
    a, b = bounds(p, g, m, v, b1, b2, t, False), bounds(p, g, m, v, b1, b2, t, True)
    for k, e in ((0, a[0] + b[0]), (2, a[1] + b[1]), (3, a[2] + b[2])):
        assert ((with_clip[k].double() - without[k].double()).abs() <= e).all()
        if exact and (k > 0 or t == 1):   # the moments always, the update while the betas' powers are exact too
            assert torch.equal(with_clip[k], without[k])
    if b2 == 0.999 and t == 7:   # the difference is there: it is what the documentation names
        assert not torch.equal(with_clip[3], without[3])
