"""The operators in the order a training step has them: residual RMSNorm, gated feed-forward block, their backward passes,
clipping and AdamW on fp32 parameters, against one float64 autograd graph; and the 8-bit pair in the order of a decode step.

End to end a value passes at most eight roundings to bf16 (norm, activation, block, and those of the backward pass), each of at
most 2^-8 of it; differences in the norm's backward pass magnify them up to four times: 2^-3 in the 2-norm. What fp32 alone
touches keeps its own bounds."""
import math

import pytest
import torch

from sirius_b200 import ops

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
BOUND = 2.0 ** -3


def rel(a, b):
    return float((a.double() - b).norm() / b.norm().clamp_min(1e-300))


@pytest.mark.parametrize("tokens,width,hidden", [(1, 64, 128), (5, 64, 136), (129, 200, 520), (700, 136, 1032), (2100, 264, 1096)])
def test_a_training_step(tokens, width, hidden):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    n = lambda *s: torch.randn(s, device="cuda", generator=g)
    x, res, dy = n(tokens, width).to(BF), n(tokens, width).to(BF), (n(tokens, width) / tokens).to(BF)
    p = {"gamma": 1 + 0.1 * n(width), "gu": 0.6 * width ** -0.5 * n(2 * hidden, width), "down": 0.6 * hidden ** -0.5 * n(width, hidden)}
    p16 = {k: p[k].to(BF) for k in ("gu", "down")}
    m, v = {k: torch.zeros_like(t) for k, t in p.items()}, {k: torch.zeros_like(t) for k, t in p.items()}
    eps, lr, steps, max_norm = 1e-6, 1e-2, 3, 0.05

    # the same step in 64 bits, from the same bf16 weights
    q = {k: t.double().clone() for k, t in p.items()}
    qm, qv = {k: torch.zeros_like(t) for k, t in q.items()}, {k: torch.zeros_like(t) for k, t in q.items()}
    for step in range(1, steps + 1):
        y, h, rstd = ops.rmsnorm(x, p["gamma"], eps, residual=res)
        out = ops.gated_ffn(y, p16["gu"], p16["down"], residual=h)
        dyn, dgu, ddown = ops.gated_ffn_backward(dy, y, p16["gu"], p16["down"], grad_dtype=torch.float32)
        dx, dgamma = ops.rmsnorm_backward(dyn, h, p["gamma"], rstd, dh=dy)
        grads = {"gamma": dgamma, "gu": dgu, "down": ddown}
        clip = ops.grad_norm(list(grads.values()), max_norm)

        leaf = {"gamma": p["gamma"].double().requires_grad_(), "gu": p16["gu"].double().requires_grad_(), "down": p16["down"].double().requires_grad_()}
        xd = x.double().requires_grad_()
        hd = xd + res.double()
        yd = hd / (hd.square().mean(-1, keepdim=True) + eps).sqrt() * leaf["gamma"]
        a, b = (yd @ leaf["gu"].T).split(hidden, 1)
        od = hd + (a * torch.sigmoid(a) * b) @ leaf["down"].T
        (od * dy.double()).sum().backward()
        assert rel(out, od.detach()) < BOUND and rel(dx, xd.grad) < BOUND
        for k in grads:
            assert rel(grads[k], leaf[k].grad) < BOUND, (step, k)
        norm = math.sqrt(sum(float(t.grad.square().sum()) for t in leaf.values()))
        assert abs(float(clip[0]) - norm) <= BOUND * norm
        own = math.sqrt(sum(float(t.double().square().sum()) for t in grads.values()))
        c = min(1.0, max_norm / (own + 1e-6))
        assert abs(float(clip[1]) - c) <= 1e-6 * c

        for k in p:
            before = p[k].double()
            ops.adamw(p[k], grads[k], m[k], v[k], lr, 0.9, 0.999, 1e-8, 0.01, step, p_bf16=p16.get(k), clip=clip)
            gc = grads[k].double() * c
            qm[k] = 0.9 * qm[k] + 0.1 * gc
            qv[k] = 0.999 * qv[k] + 0.001 * gc * gc
            up = lr / (1 - 0.9 ** step) * qm[k] / ((qv[k] / (1 - 0.999 ** step)).sqrt() + 1e-8)
            # fp32 moments of earlier steps included: 64 roundings of 2^-24, magnified where the moments cancel
            assert ((p[k].double() - (before * (1 - lr * 0.01) - up)).abs() <= 4e-7 * before.abs() + 1e-5 * lr + 1e-5 * up.abs()).all(), (step, k)
            if k in p16:
                assert torch.equal(p16[k], p[k].to(BF))
    assert ops.tc_status() == 0


@pytest.mark.parametrize("tokens,width,hidden", [(1, 64, 128), (3, 512, 1024), (24, 1040, 2008), (300, 272, 1032)])
def test_a_decode_step_in_8_bits(tokens, width, hidden):
    """Both operands of the projections are rounded to e4m3, each by at most 2^-4 of a value (or of 2^-6 of a row's largest):
    gate and up are off by at most 2^-3 in the 2-norm, their product by 2^-2."""
    g = torch.Generator(device="cuda").manual_seed(tokens)
    n = lambda *s: torch.randn(s, device="cuda", generator=g)
    x, res, gamma = n(tokens, width).to(BF), n(tokens, width).to(BF), 1 + 0.1 * n(width)
    wgu, wd = (0.6 * width ** -0.5 * n(2 * hidden, width)).to(BF), (0.6 * hidden ** -0.5 * n(width, hidden)).to(BF)
    wq, ws = ops.quantize_rows_e4m3(wgu)
    q, scale, h, _ = ops.rmsnorm_e4m3(x, gamma, 1e-6, residual=res)
    y = ops.gated_ffn_e4m3(q, scale, wq, ws, wd, residual=h)
    hd = x.double() + res.double()
    yd = hd / (hd.square().mean(-1, keepdim=True) + 1e-6).sqrt() * gamma.double()
    a, b = (yd @ wgu.double().T).split(hidden, 1)
    ffn = (a * torch.sigmoid(a) * b) @ wd.double().T
    got = y.double() - h.double()
    assert float((got - ffn).norm()) <= 0.25 * float(ffn.norm()) + 2.0 ** -8 * float(y.double().norm()) + 2.0 ** -8 * float(hd.norm())
    # from the 8-bit operands themselves the block is as exact as its bf16 form
    a, b = ((q.double() * scale.double()[:, None]) @ (wq.double() * ws.double()[:, None]).T).split(hidden, 1)
    want = h.double() + (a * torch.sigmoid(a) * b) @ wd.double().T
    assert rel(y, want) < 2.0 ** -7
    assert ops.tc_status() == 0
