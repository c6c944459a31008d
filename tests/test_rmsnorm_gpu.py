"""Residual RMSNorm, its e4m3 output and its backward pass against the definitions in 64 bits.

Tolerances: a row's statistic adds at most 32 squares a lane, then 5 shuffles and 15 warps, in fp32: within 53 steps of 2^-24,
halved by the root; with the roundings of the sum, the root (2^-22) and the products all fp32 results are within 64 x 2^-24.
Results in bf16 are rounded once more, by at most 2^-8; in e4m3 by 2^-4, or half the smallest step, 2^-10 of the scale."""
import pytest
import torch

from sirius_b200 import ops

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24
EPS = 1e-6
# rows, columns: one row; a vector; lanes without a vector; one to sixteen warps a row; the longest rows of either type
SIZES = [(1, 8), (1, 896), (3, 24), (5, 264), (8, 1024), (1, 4096), (24, 4096), (777, 2056), (1500, 896), (5000, 72), (33, 8192), (700, 8192)]


def make(rows, c, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 100 * rows + c)
    n = lambda *s: torch.randn(s, device="cuda", generator=g)
    return {"x": (n(rows, c) * 2).to(dtype), "res": n(rows, c).to(dtype), "gamma": 1 + 0.2 * n(c), "dy": n(rows, c).to(dtype), "dh": n(rows, c).to(dtype)}


def half(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, tol, what):
    d = (got.double() - want).abs()
    assert (d <= tol + 1e-40).all(), f"{what}: off by up to {float((d - tol).max()):.3g} beyond the bound"


def norm64(s, residual):
    h = s["x"].double() + (s["res"].double() if residual else 0)
    r = 1 / (h.square().mean(-1) + EPS).sqrt()
    return h, r, h * r[:, None] * s["gamma"].double()


@pytest.mark.parametrize("rows,c", SIZES + [(3, 16384)])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("residual", [True, False])
def test_forward(rows, c, dtype, residual):
    if c > 8192 and dtype == F32:
        pytest.skip("a row of 32 KB is the longest")
    s = make(rows, c, dtype)
    y, h, rstd = ops.rmsnorm(s["x"], s["gamma"], EPS, residual=s["res"] if residual else None)
    h64, r64, y64 = norm64(s, residual)
    close(rstd, r64, 64 * U * r64, "rstd")
    close(y, y64, (64 * U + half(dtype)) * 1.01 * y64.abs(), "y")
    close(h, h64, (half(dtype) + U) * 1.01 * h64.abs(), "h")
    assert (h is s["x"]) == (not residual)


@pytest.mark.parametrize("rows,c", SIZES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_e4m3_output(rows, c, dtype):
    s = make(rows, c, dtype)
    q, scale, h, rstd = ops.rmsnorm_e4m3(s["x"], s["gamma"], EPS, residual=s["res"])
    h64, r64, y64 = norm64(s, True)
    s64 = y64.abs().amax(-1) / 448
    close(scale, s64, 64 * U * s64, "scale")
    close(rstd, r64, 64 * U * r64, "rstd")
    close(h, h64, (half(dtype) + U) * 1.01 * h64.abs(), "h")
    close(q.double() * scale.double()[:, None], y64, torch.maximum(2.0 ** -4 * y64.abs(), 2.0 ** -10 * s64[:, None]) * (1 + 2.0 ** -10), "q")
    assert (q.float().abs().amax(-1) == 448).all()


@pytest.mark.parametrize("rows,c", SIZES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_quantised_rows(rows, c, dtype):
    s = make(rows, c, dtype)
    q, scale = ops.quantize_rows_e4m3(s["x"])
    x64 = s["x"].double()
    s64 = x64.abs().amax(-1) / 448
    close(scale, s64, 2 * U * s64, "scale")
    close(q.double() * scale.double()[:, None], x64, torch.maximum(2.0 ** -4 * x64.abs(), 2.0 ** -10 * s64[:, None]) * (1 + 2.0 ** -10), "q")


@pytest.mark.parametrize("rows,c", SIZES)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("with_dh", [True, False])
def test_backward(rows, c, dtype, with_dh):
    s = make(rows, c, dtype)
    rstd = (1 / (s["x"].double().square().mean(-1) + EPS).sqrt()).float()
    dx, dgamma = ops.rmsnorm_backward(s["dy"], s["x"], s["gamma"], rstd, dh=s["dh"] if with_dh else None)
    r, x, dy, gamma = rstd.double()[:, None], s["x"].double(), s["dy"].double(), s["gamma"].double()
    dh = s["dh"].double() if with_dh else torch.zeros_like(x)
    xhat, g = x * r, dy * gamma
    want = dh + r * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    terms = dh.abs() + r * (g.abs() + xhat.abs() * (g * xhat).abs().mean(-1, keepdim=True))
    close(dx, want, half(dtype) * want.abs() + 64 * U * terms, "dx")
    p = dy * xhat
    close(dgamma, p.sum(0), (rows + 64) * U * p.abs().sum(0), "dgamma")
    again = ops.rmsnorm_backward(s["dy"], s["x"], s["gamma"], rstd, dh=s["dh"] if with_dh else None)
    assert torch.equal(dx, again[0]) and torch.equal(dgamma, again[1])


def test_backward_against_differences():
    s = make(40, 264, F32)
    eps = 1e-2
    y, h, rstd = ops.rmsnorm(s["x"], s["gamma"], eps, residual=s["res"])
    dx, dgamma = ops.rmsnorm_backward(s["dy"], h, s["gamma"], rstd, dh=s["dh"])
    dy, dh = s["dy"].double(), s["dh"].double()

    def loss(x, gamma):
        hh = x + s["res"].double()
        return (dy * gamma * hh / (hh.square().mean(-1, keepdim=True) + eps).sqrt()).sum() + (dh * hh).sum()
    x, gamma = s["x"].double(), s["gamma"].double()
    gen = torch.Generator(device="cuda").manual_seed(3)
    for which, got in ((0, dx), (1, dgamma)):
        d = torch.randn(got.shape, device="cuda", dtype=torch.float64, generator=gen)
        t = 1e-5
        a, b = ((x + t * d, gamma), (x - t * d, gamma)) if which == 0 else ((x, gamma + t * d), (x, gamma - t * d))
        slope = (loss(*a) - loss(*b)) / (2 * t)
        # fp32 results: 128 x 2^-24 of their magnitude and that of what cancels in them, the differences 1e-8 of the terms
        assert ((got.double() * d).sum() - slope).abs() <= (256 * U + 1e-8) * (got.double().abs() * d.abs()).sum() + 256 * U * d.abs().sum() * 4


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_with_nothing_and_with_nan(dtype):
    s = make(9, 264, dtype)
    x = s["x"].clone()
    x[2] = 0
    x[4, 7] = float("nan")
    x[6, 3] = float("inf")
    y, _, _ = ops.rmsnorm(x, s["gamma"], EPS)
    q, scale, _, _ = ops.rmsnorm_e4m3(x, s["gamma"], EPS)
    p, pscale = ops.quantize_rows_e4m3(x)
    good = [0, 1, 3, 5, 7, 8]
    assert torch.equal(y[good], ops.rmsnorm(s["x"], s["gamma"], EPS)[0][good])
    assert (y[2] == 0).all() and (q[2].float() == 0).all() and (p[2].float() == 0).all() and scale[2] == 2.0 ** -126 and pscale[2] == 2.0 ** -126
    assert y[4].isnan().all() and scale[4].isnan() and q[4].float().isnan().all() and pscale[4].isnan() and p[4].float().isnan().all()
    assert y[6, 3].isnan() and (y[6, 4:] == 0).all() and scale[6].isnan() and pscale[6].isinf()
    assert torch.isfinite(scale[good]).all() and torch.isfinite(q[good].float()).all()


def test_in_place_and_no_rows():
    from sirius_b200._lib import SRT_BF16, call
    s = make(50, 896, BF)
    y, h, rstd = ops.rmsnorm(s["x"], s["gamma"], EPS, residual=s["res"])
    x, y2, st = s["x"].clone(), torch.empty_like(y), torch.cuda.current_stream().cuda_stream
    call("srt_rmsnorm_fwd", SRT_BF16, s["res"].data_ptr(), x.data_ptr(), s["gamma"].data_ptr(), x.data_ptr(), y2.data_ptr(), None, 50, 896, EPS, st)
    assert torch.equal(x, h) and torch.equal(y2, y)
    e = s["x"][:0]
    assert ops.rmsnorm(e, s["gamma"], EPS)[0].shape == (0, 896)
    dx, dgamma = ops.rmsnorm_backward(e, e, s["gamma"], rstd[:0])
    assert dx.shape == (0, 896) and not dgamma.any()


def test_leading_axes_and_other_stream():
    s = make(60, 264, BF)
    want = ops.rmsnorm(s["x"], s["gamma"], EPS, residual=s["res"])
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = ops.rmsnorm(s["x"].view(3, 20, 264), s["gamma"], EPS, residual=s["res"].view(3, 20, 264))
    torch.cuda.synchronize()
    assert got[2].shape == (3, 20)
    for a, b in zip(got, want):
        assert torch.equal(a.reshape(b.shape), b)
