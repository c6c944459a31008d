"""The operators where offsets pass 32 bits, and shapes at the edge of what they take: rows and lists of more than 2^31 elements, the
widest 8-bit rows, one row without a leading axis, a first call inside a capture. Large results are looked at in rows from the
beginning, the middle and the end, against 64 bits.

Tolerances as in the operators' own tests: fp32 statistics and products within 64 x 2^-24, results rounded once more to their
type (bf16 2^-8, e4m3 2^-4 or 2^-10 of the scale); sums over n rows within (n + 64) 2^-24 of their magnitudes."""
import subprocess
import sys

import pytest
import torch
from test_gated_ffn_gpu import H, close, reference

from sirius_b200 import ops

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def filled(*shape, seed, std=1.0):
    """bf16 draws made in pieces, so that no fp32 copy of the whole is needed."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = torch.empty(shape, device="cuda", dtype=BF)
    for piece in out.view(-1).split(1 << 28):
        piece.normal_(0.0, std, generator=g)
    return out


def test_norms_of_more_than_2_to_31_elements():
    rows, c = 264007, 8192   # 2.16 G elements
    x, gamma = filled(rows, c, seed=1, std=2.0), torch.linspace(0.5, 1.5, c, device="cuda")
    pick = torch.tensor([0, 1, 131071, 262143, 262144, rows - 2, rows - 1], device="cuda")
    x64 = x[pick].double()
    r64 = 1 / (x64.square().mean(-1) + 1e-6).sqrt()
    y64 = x64 * r64[:, None] * gamma.double()
    y, h, rstd = ops.rmsnorm(x, gamma, 1e-6)
    assert h is x and ((rstd[pick].double() - r64).abs() <= 64 * U * r64).all()
    assert ((y[pick].double() - y64).abs() <= (64 * U + H) * 1.01 * y64.abs()).all()
    del y
    q, scale = ops.quantize_rows_e4m3(x)
    s64 = x64.abs().amax(-1) / 448
    assert ((scale[pick].double() - s64).abs() <= 2 * U * s64).all()
    bound = torch.maximum(2.0 ** -4 * x64.abs(), 2.0 ** -10 * s64[:, None]) * (1 + 2.0 ** -10)
    assert ((q[pick].double() * scale[pick].double()[:, None] - x64).abs() <= bound).all()
    del q
    dy = filled(rows, c, seed=2)
    dx, dgamma = ops.rmsnorm_backward(dy, x, gamma, rstd)
    r, d = rstd[pick].double()[:, None], dy[pick].double()
    xhat, g = x64 * r, d * gamma.double()
    want = r * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    terms = r * (g.abs() + xhat.abs() * (g * xhat).abs().mean(-1, keepdim=True))
    assert ((dx[pick].double() - want).abs() <= H * want.abs() + 64 * U * terms).all()
    total, size = torch.zeros(c, device="cuda", dtype=torch.float64), torch.zeros(c, device="cuda", dtype=torch.float64)
    for a in range(0, rows, 16384):
        p = dy[a:a + 16384].double() * x[a:a + 16384].double() * rstd[a:a + 16384].double()[:, None]
        total += p.sum(0)
        size += p.abs().sum(0)
    assert ((dgamma.double() - total).abs() <= (rows + 64) * U * size).all()


def test_gradients_of_more_than_2_to_31_elements():
    n = (1 << 31) + 12347
    flat = filled(n + 3, seed=3, std=1e-3)
    grads = [flat[:5], flat[5:n], flat[n:]]   # the long one begins off a vector boundary and ends inside one
    picks = [flat[a:a + 100].clone() for a in (0, (1 << 31) - 50, n - 97)]
    norm = float(sum(p.double().square().sum() for p in flat.split(1 << 26)).sqrt())
    clip = ops.clip_grad_norm(grads, norm / 8)
    c = 0.125 * norm / (norm + 1e-6)
    assert abs(float(clip[0]) - norm) <= 2 * U * norm and abs(float(clip[1]) - c) <= 2 * U * c
    for a, before in zip((0, (1 << 31) - 50, n - 97), picks):
        want = before.double() * c
        assert ((flat[a:a + 100].double() - want).abs() <= (H + 3 * U) * want.abs()).all()


def test_a_block_close_to_2_to_31_elements():
    t, c, f = 220000, 896, 4864   # tokens x 2 hidden = 2.14 G elements
    x, dy = filled(t, c, seed=4), filled(t, c, seed=5)
    wgu, wd = filled(2 * f, c, seed=6, std=0.7 * c ** -0.5), filled(c, f, seed=7, std=0.7 * f ** -0.5)
    pick = torch.tensor([0, 127, 128, 109999, 110000, t - 2, t - 1], device="cuda")
    y = ops.gated_ffn(x, wgu, wd, residual=dy)
    assert ops.tc_status() == 0
    close(y[pick], *reference(x[pick], wgu, wd, dy[pick]), "y")
    del y
    dx, dwgu, dwd = ops.gated_ffn_backward(dy, x, wgu, wd, grad_dtype=F32)
    assert ops.tc_status() == 0
    want, tol = reference(x[pick], wgu, wd, dy=dy[pick])
    close(dx[pick], want[0], (tol[0] + H * (want[0].abs() + tol[0])) * 1.01, "dx")
    # the weights' gradients of a few hidden channels, over all tokens
    channels = torch.tensor([0, 1, 2431, f - 1], device="cuda")
    rows = torch.cat([channels, f + channels])
    dw, ew, dd, ed = 0, 0, 0, 0
    for a in range(0, t, 20000):
        xs, ds = x[a:a + 20000].double(), dy[a:a + 20000].double()
        g, u = xs @ wgu[channels].double().T, xs @ wgu[f + channels].double().T
        eg, eu = (c * 2.0 ** -23 * (xs.abs() @ w.double().abs().T) for w in (wgu[channels], wgu[f + channels]))
        s = torch.sigmoid(g)
        da = ds @ wd[:, channels].double()
        ea = c * 2.0 ** -23 * (ds.abs() @ wd[:, channels].double().abs())
        act = g * s * u
        dgu = torch.cat([da * u * s * (1 + g * (1 - s)), da * g * s], 1)
        # gate, up and da to fp32, the sigmoid 2^-18, the rounding of the operand 2^-8
        e_act = H * act.abs() + 1.01 * (1.1 * u.abs() * eg + (g * s).abs() * eu + 2.0 ** -18 * act.abs())
        e_gate = 1.1 * u.abs() * ea + 1.1 * da.abs() * eu + 0.5 * (da * u).abs() * eg + 2.0 ** -18 * 1.1 * (da * u).abs()
        e_up = (g * s).abs() * ea + 1.1 * da.abs() * eg + 2.0 ** -18 * (da * g * s).abs()
        e_dgu = H * dgu.abs() + 1.01 * torch.cat([e_gate, e_up], 1)
        dw, ew = dw + dgu.T @ xs, ew + (e_dgu + t * 2.0 ** -23 * dgu.abs()).T @ xs.abs()
        dd, ed = dd + ds.T @ act, ed + ds.abs().T @ (e_act + t * 2.0 ** -23 * act.abs())
    close(dwgu[rows], dw, ew * 1.01 + 2.0 ** -23 * dw.abs(), "dw_gate_up")
    close(dwd[:, channels], dd, ed * 1.01 + 2.0 ** -23 * dd.abs(), "dw_down")


@pytest.mark.parametrize("dtype,c", [(BF, 8200), (BF, 12288), (BF, 16384), (F32, 4104), (F32, 8192)])
@pytest.mark.parametrize("rows", [1, 300])
def test_the_widest_8_bit_rows(dtype, c, rows):
    g = torch.Generator(device="cuda").manual_seed(c + rows)
    x, res = ((torch.randn(rows, c, device="cuda", generator=g) * 2).to(dtype) for _ in range(2))
    gamma = 1 + 0.2 * torch.randn(c, device="cuda", generator=g)
    q, scale, h, rstd = ops.rmsnorm_e4m3(x, gamma, 1e-6, residual=res)
    h64 = x.double() + res.double()
    y64 = h64 / (h64.square().mean(-1, keepdim=True) + 1e-6).sqrt() * gamma.double()
    s64 = y64.abs().amax(-1) / 448
    assert ((scale.double() - s64).abs() <= 64 * U * s64).all()
    assert ((h.double() - h64).abs() <= (torch.finfo(dtype).eps / 2 + U) * 1.01 * h64.abs()).all()
    bound = torch.maximum(2.0 ** -4 * y64.abs(), 2.0 ** -10 * s64[:, None]) * (1 + 2.0 ** -10)
    assert ((q.double() * scale.double()[:, None] - y64).abs() <= bound).all()
    p, pscale = ops.quantize_rows_e4m3(x)
    p64 = x.double().abs().amax(-1) / 448
    bound = torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * p64[:, None]) * (1 + 2.0 ** -10)
    assert ((p.double() * pscale.double()[:, None] - x.double()).abs() <= bound).all()


def test_one_row_without_a_leading_axis():
    x, gamma = torch.randn(896, device="cuda").to(BF), torch.ones(896, device="cuda")
    y, h, rstd = ops.rmsnorm(x, gamma)
    q, scale = ops.quantize_rows_e4m3(x)
    dx, dgamma = ops.rmsnorm_backward(x, x, gamma, rstd)
    y2, _, rstd2 = ops.rmsnorm(x[None], gamma)
    dx2, dgamma2 = ops.rmsnorm_backward(x[None], x[None], gamma, rstd2)
    assert y.shape == (896,) and rstd.shape == () and scale.shape == () and q.shape == (896,)
    assert torch.equal(y, y2[0]) and torch.equal(dx, dx2[0]) and torch.equal(dgamma, dgamma2)


FIRST = """
import torch
from sirius_b200 import ops
BF = torch.bfloat16
x, wgu, wd = torch.randn(600, 136, device="cuda").to(BF), torch.randn(528, 136, device="cuda").to(BF), torch.randn(136, 264, device="cuda").to(BF)
gamma, grads = torch.ones(136, device="cuda"), [torch.randn(1000, device="cuda") for _ in range(40)]
def calls():
    y, h, rstd = ops.rmsnorm(x, gamma, residual=x)
    return (y, rstd, ops.gated_ffn(y, wgu, wd, h), ops.gated_ffn(x[:1], wgu, wd), *ops.gated_ffn_backward(x, y, wgu, wd),
            *ops.rmsnorm_backward(x, h, gamma, rstd), ops.grad_norm(grads, 1.0))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = calls()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, calls())) and ops.tc_status() == 0
"""


def test_the_first_call_of_a_process_may_be_captured():
    r = subprocess.run([sys.executable, "-c", FIRST], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
