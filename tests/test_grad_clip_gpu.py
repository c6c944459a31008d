"""Global gradient norm, clipping in place, and the optimizer steps that take the coefficient, against 64 bits.

Tolerances: norm and coefficient are rounded once from 64 bits (2^-24); a clipped gradient is a product of fp32 values, rounded
once more (fp32 2^-24, bf16 2^-8)."""
import math

import pytest
import torch

from sirius_b200 import ops

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24

LISTS = [[1], [3], [32768], [32769], [7, 1, 65537, 12], [100000] * 5, [5] * 33, [17, 0, 4099] * 30, [33] * 1024, [19] * 1025, [3001] * 2100]


def make(sizes, dtype, seed=0, packed=True):
    """Tensors back to back in one buffer, so that most begin off a 16-byte boundary, between two guard regions."""
    g = torch.Generator(device="cuda").manual_seed(seed + len(sizes))
    flat = torch.randn(sum(sizes) + 16, device="cuda", generator=g).to(dtype)
    at, out = 8, []
    for n in sizes:
        out.append(flat[at:at + n])
        at += n
    return flat, out


@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("share", [0.3, 5.0])
def test_norm_and_clip(sizes, dtype, share):
    flat, grads = make(sizes, dtype)
    before = flat.clone()
    norm = float(before[8:-8].double().square().sum().sqrt())
    max_norm = share * norm
    c = min(1.0, max_norm / (norm + 1e-6))
    clip = ops.grad_norm(grads, max_norm)
    assert torch.equal(flat, before)
    assert abs(float(clip[0]) - norm) <= 2 * U * norm and abs(float(clip[1]) - c) <= 2 * U * c
    got = ops.clip_grad_norm(grads, max_norm)
    assert torch.equal(got, clip)
    assert torch.equal(flat[:8], before[:8]) and torch.equal(flat[-8:], before[-8:])
    want = before[8:-8].double() * c
    half = 2.0 ** -8 if dtype == BF else U
    assert ((flat[8:-8].double() - want).abs() <= (half + 3 * U) * want.abs()).all()


def test_many_elements():
    """More chunks than blocks, and a tensor of 2^27 elements; the parts of the sum meet in 64 bits."""
    flat, grads = make([1 << 27, 999, 1 << 24], F32)
    norm = float(torch.linalg.vector_norm(flat[8:-8].double()))
    clip = ops.clip_grad_norm(grads, 1.0)
    assert abs(float(clip[0]) - norm) <= 2 * U * norm
    again = float(torch.linalg.vector_norm(flat[8:-8].double()))
    assert abs(again - norm / (norm + 1e-6)) <= 4 * U


def test_values_whose_squares_do_not_fit_fp32():
    g = torch.full((1000,), 1e30, device="cuda")
    clip = ops.clip_grad_norm([g], 2.0)
    n = float(torch.tensor(1e30)) * math.sqrt(1000)
    assert abs(float(clip[0]) - n) <= 2 * U * n and torch.isfinite(g).all() and abs(float(g.double().norm()) - 2.0) < 1e-5
    g = torch.full((1000,), 1e-30, device="cuda")
    assert abs(float(ops.grad_norm([g], 1.0)[0]) - 1e-30 * math.sqrt(1000)) <= 4 * U * 1e-28 and float(ops.grad_norm([g], 1.0)[1]) == 1.0


def test_not_a_number_and_infinity_are_not_hidden():
    for bad in (float("nan"), float("inf")):
        _, grads = make([100, 7, 3000], F32)
        grads[1][3] = bad
        clip = ops.clip_grad_norm(grads, 1.0)
        if math.isnan(bad):
            assert clip.isnan().all() and all(g.isnan().all() for g in grads)
        else:
            assert clip[0].isinf() and clip[1] == 0 and grads[1][3].isnan() and (grads[0] == 0).all()


def test_nothing_to_clip():
    empty = torch.empty(0, device="cuda")
    for grads in ([], [empty], [empty, empty]):
        for f in (ops.grad_norm, ops.clip_grad_norm):
            assert f(grads, 1.0).tolist() == [0.0, 1.0]


def test_tensors_that_share_memory():
    from sirius_b200._lib import SrtError
    flat = torch.randn(1000, device="cuda")
    before = flat.clone()
    for grads in ([flat[:600], flat[500:]], [flat[700:], flat[:300], flat[200:500]], [flat, flat], [flat[10:20], flat[5:11]]):
        with pytest.raises(SrtError, match="shares memory"):
            ops.clip_grad_norm(grads, 1e-3)
        assert torch.equal(flat, before)
        assert torch.isfinite(ops.grad_norm(grads, 1.0)).all()
    for grads in ([flat[500:], flat[:500]], [flat[10:20], flat[:0], flat[:10], flat[20:]], [flat[20:], flat[10:10], flat[:20]]):
        flat.copy_(before)
        ops.clip_grad_norm(grads, 1e-3)
        assert abs(float(flat.double().norm()) - 1e-3) < 1e-6


def test_an_empty_step():
    e = torch.empty(0, device="cuda")
    clip = ops.grad_norm([], 1.0)
    ops.adamw(e, e, e, e, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, clip=clip)
    ops.sgd_momentum(e, e, e, 1e-3, 0.9, 0.0, True, clip=clip)


@pytest.mark.parametrize("n", [1, 5, 1000, 100003, 1 << 20])
@pytest.mark.parametrize("share", [0.25, 4.0])
def test_adamw_takes_the_coefficient(n, share):
    g = torch.Generator(device="cuda").manual_seed(n)
    r = lambda s: torch.randn(n, device="cuda", generator=g) * s
    p, gr, m, v = r(0.05), r(1e-2), r(1e-3), r(1e-2).square()
    pb = torch.empty(n, device="cuda", dtype=BF)
    lr, b1, b2, eps, wd, step = 3e-4, 0.9, 0.999, 1e-8, 0.01, 7
    norm = float(gr.double().norm())
    c = min(1.0, share * norm / (norm + 1e-6))
    p0, g0, m0, v0 = (t.double() for t in (p, gr.clone(), m, v))
    clip = ops.grad_norm([gr], share * norm)
    ops.adamw(p, gr, m, v, lr, b1, b2, eps, wd, step, p_bf16=pb, clip=clip)
    assert torch.equal(gr.double(), g0)
    gc = g0 * c
    m1, v1 = b1 * m0 + (1 - b1) * gc, b2 * v0 + (1 - b2) * gc * gc
    up = lr / (1 - b1 ** step) * m1 / (v1.sqrt() / math.sqrt(1 - b2 ** step) + eps)
    p1 = p0 * (1 - lr * wd) - up
    # every fp32 operation and constant is within 2^-24: at most eight on the way to m and v, sixteen more to the update
    em = 8 * U * (b1 * m0.abs() + (1 - b1) * gc.abs())
    assert ((m.double() - m1).abs() <= em).all()
    assert ((v.double() - v1).abs() <= 10 * U * v1).all()
    scale = lr / (1 - b1 ** step) / (v1.sqrt() / math.sqrt(1 - b2 ** step) + eps)
    assert ((p.double() - p1).abs() <= 4 * U * p0.abs() + 32 * U * up.abs() + em * scale).all()
    assert torch.equal(pb, p.to(BF))


@pytest.mark.parametrize("first", [True, False])
def test_sgd_takes_the_coefficient(first):
    n = 10007
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda s: torch.randn(n, device="cuda", generator=g) * s
    p, gr, m = r(0.05), r(1e-2), r(1e-3)
    p0, m0 = p.double(), m.double()
    clip = ops.grad_norm([gr], 0.1)
    c = 0.1 / (float(gr.double().norm()) + 1e-6)
    ops.sgd_momentum(p, gr, m, 0.1, 0.9, 1e-4, first, clip=clip)
    d = 1e-4 * p0 + gr.double() * c
    m1 = d if first else 0.9 * m0 + d
    e = 8 * U * (1e-4 * p0.abs() + (gr.double() * c).abs() + (0 if first else 0.9 * m0.abs()))
    assert ((m.double() - m1).abs() <= e).all()
    assert ((p.double() - (p0 - 0.1 * m1)).abs() <= 4 * U * p0.abs() + 0.1 * e + 4 * U * 0.1 * m1.abs()).all()


def test_a_coefficient_of_one_changes_no_bit():
    n = 4099
    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda s: torch.randn(n, device="cuda", generator=g) * s
    a = [r(0.05), r(1e-2), r(1e-3)]
    b = [t.clone() for t in a]
    ops.sgd_momentum(*a, 0.1, 0.9, 1e-4, False)
    ops.sgd_momentum(*b, 0.1, 0.9, 1e-4, False, clip=ops.grad_norm([b[1]], 1e6))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_lists_of_many_tensors():
    flat, grads = make([999] * 1500, F32)
    start = flat.clone()
    want = ops.clip_grad_norm(grads, 3.0).clone()
    clipped = flat.clone()
    flat.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        clip = ops.clip_grad_norm(grads, 3.0)
    for _ in range(2):
        flat.copy_(start)
        graph.replay()
        assert torch.equal(clip, want) and torch.equal(flat, clipped)


@pytest.mark.parametrize("n", [5, 4099, 300001])
def test_steps_on_views_off_a_vector_boundary(n):
    """Views that begin at any element take the same step as copies of them that begin on a boundary."""
    g = torch.Generator(device="cuda").manual_seed(n)
    for shift in (1, 2, 3):
        flat = [torch.randn(n + 4, device="cuda", generator=g).square() * 0.01 for _ in range(4)]
        views, copies = [t[shift:shift + n] for t in flat], [t[shift:shift + n].clone() for t in flat]
        outside = [t.clone() for t in flat]
        low = [torch.empty(n + 4, device="cuda", dtype=BF)[shift:shift + n], torch.empty(n, device="cuda", dtype=BF)]
        clip = ops.grad_norm([views[1]], 0.5)
        for k, t in enumerate((views, copies)):
            ops.sgd_momentum(*t[:3], 0.1, 0.9, 1e-4, False, p_bf16=low[k], clip=clip)
        assert torch.equal(*low)
        for k, t in enumerate((views, copies)):
            ops.adamw(*t, 1e-3, 0.9, 0.99, 1e-8, 0.01, 3, p_bf16=low[k], clip=clip)
        assert torch.equal(*low) and all(torch.equal(a, b) for a, b in zip(views, copies))
        for t, o in zip(flat, outside):
            assert torch.equal(t[:shift], o[:shift]) and torch.equal(t[shift + n:], o[shift + n:])


@pytest.mark.parametrize("n", [1000, 100003])
def test_adamw_keeps_its_roundings(n):
    """m = fma(1 - b1, g, b1 m), v = fma((1 - b2) g, g, b2 v): with g, m and v of eight bits the sums below are exact in 64 bits,
    so one rounding is left in each. With or without a coefficient of one, the bits are the same."""
    g = torch.Generator(device="cuda").manual_seed(n)
    r = lambda s: (torch.randn(n, device="cuda", generator=g) * s).to(BF).float()
    p, gr, m, v = r(0.05), r(1e-2), r(1e-3), r(1e-2).square().to(BF).float()
    b1, b2 = 0.875, 0.9375
    c1, c2 = 1 - b1, 1 - b2
    want_m = (c1 * gr.double() + (b1 * m).double()).float()
    want_v = ((c2 * gr).double() * gr.double() + (b2 * v).double()).float()
    a, b = ([t.clone() for t in (p, gr, m, v)] for _ in range(2))
    ops.adamw(*a, 2.0 ** -10, b1, b2, 2.0 ** -27, 0.0, 1)
    ops.adamw(*b, 2.0 ** -10, b1, b2, 2.0 ** -27, 0.0, 1, clip=ops.grad_norm([b[1]], 1e6))
    assert torch.equal(a[2], want_m) and torch.equal(a[3], want_v)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
