"""RMSNorm backward on the longest rows, around every change of its launch: sixteen warps a row with two, three and four
vectors a lane, and the widths whose columns of dgamma fill the shared memory that a kernel has without asking for more.

Tolerances as in the other widths: fp32 results within 64 x 2^-24 of the magnitudes that meet in them (a row's statistic adds at
most 32 products a lane, then 5 shuffles and 15 warps), dx rounded once more to its type, dgamma a sum over the rows."""
import pytest
import torch

from sirius_b200 import ops

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def compare(rows, c, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows + c)
    n = lambda *s: torch.randn(s, device="cuda", generator=g)
    h, dy, dh, gamma = (n(rows, c) * 2).to(dtype), n(rows, c).to(dtype), n(rows, c).to(dtype), 1 + 0.2 * n(c)
    rstd = (1 / (h.double().square().mean(-1) + 1e-6).sqrt()).float()
    dx, dgamma = ops.rmsnorm_backward(dy, h, gamma, rstd, dh=dh)
    r, x, d = rstd.double()[:, None], h.double(), dy.double()
    xhat, gd = x * r, d * gamma.double()
    want = dh.double() + r * (gd - xhat * (gd * xhat).mean(-1, keepdim=True))
    terms = dh.double().abs() + r * (gd.abs() + xhat.abs() * (gd * xhat).abs().mean(-1, keepdim=True))
    assert ((dx.double() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + 64 * U * terms).all()
    p = d * xhat
    assert ((dgamma.double() - p.sum(0)).abs() <= (rows + 64) * U * p.abs().sum(0)).all()
    again = ops.rmsnorm_backward(dy, h, gamma, rstd, dh=dh)
    assert torch.equal(dx, again[0]) and torch.equal(dgamma, again[1])


@pytest.mark.parametrize("c", [8192, 8200, 12224, 12232, 12280, 12288, 12296, 16376, 16384])
@pytest.mark.parametrize("rows", [1, 300])
def test_bf16_rows(rows, c):
    compare(rows, c, BF)


@pytest.mark.parametrize("c", [4096, 4104, 6144, 6152, 8184, 8192])
@pytest.mark.parametrize("rows", [1, 300])
def test_fp32_rows(rows, c):
    compare(rows, c, F32)
