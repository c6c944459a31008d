"""clip_grad_norm of the four executors: the norm is that of the gradients they report, the next optimizer step takes the
coefficient (seen in the first moment, which is linear in the gradient), and a later forward_backward takes it back.

Tolerances: the norm is a sum in 64 bits of what `get` reports, rounded once (2^-24), the reported gradients are exact copies;
a moment is four fp32 operations on values of its own size (8 x 2^-24 of their magnitudes)."""
import math

import numpy as np
import pytest
import torch

from sirius_b200 import ops
from sirius_b200.gpt2_step import Gpt2Step
from sirius_b200.qwen2_step import Qwen2Step
from sirius_b200.step import GET_GRAD, GET_MOMENTUM, ResNetStep
from sirius_b200.swin_step import SwinStep

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def gpt2():
    s = Gpt2Step(n_layer=2, n_head=2, d_model=128, vocab=311, ctx=64, max_batch=2, seq=64)
    rng = np.random.default_rng(0)
    s.load_state_dict({n: rng.normal(0, 0.02, sh).astype(np.float32) for n, (_, sh) in s.params.items()})
    s.upload_tokens(rng.integers(0, 311, (2, 64)))
    return s, lambda: s.forward_backward(), "adamw"


def qwen2():
    s = Qwen2Step(n_layer=2, n_head=4, n_kv_head=2, hidden=128, intermediate=256, vocab=500, max_batch=2, seq=128)
    rng = np.random.default_rng(1)
    s.load_state_dict({n: (1 if sh == (128,) and "norm" in n else 0) + rng.normal(0, 0.02, sh).astype(np.float32) for n, (_, sh) in s.params.items()})
    s.upload_tokens(rng.integers(0, 500, (2, 128)))
    return s, lambda: s.forward_backward(), "adamw"


def swin():
    s = SwinStep(image=224, patch=4, embed=32, depths=(2, 2, 2, 2), heads=(2, 4, 8, 16), window=7, num_classes=40, max_batch=2)
    rng = np.random.default_rng(2)
    s.load_state_dict({n: (1 if "norm" in n and n.endswith("weight") else 0) + rng.normal(0, 0.02, sh).astype(np.float32) for n, (_, sh) in s.params.items()})
    g = torch.Generator().manual_seed(2)
    s.upload_batch(torch.randn(2, 3, 224, 224, generator=g), torch.randint(0, 40, (2,), generator=g))
    return s, lambda: s.forward_backward(), "adamw"


def resnet():
    from oracle import resnet_oracle as O
    s = ResNetStep(layers=O.LAYERS["resnet14"], max_batch=4, image=64, dtype="bf16")
    s.load_state_dict(O.state_arrays(O.build_model("resnet14", 0)))
    s.upload_batch(*O.make_batches(4, 1, 64)[0])
    return s, lambda: s.forward_backward(4, 4), "sgd"


def norm_of(grads):
    return math.sqrt(sum(float(np.sum(np.square(g.astype(np.float64)))) for g in grads.values()))


@pytest.mark.parametrize("make", [gpt2, qwen2, swin, resnet], ids=lambda f: f.__name__)
@pytest.mark.parametrize("share", [0.25, 3.0])
def test_the_next_step_takes_the_coefficient(make, share):
    s, backward, kind = make()
    names = [n for n in s.params if "running" not in n]
    try:
        backward()
        grads = {n: s.get(n, GET_GRAD) for n in names}
        norm = norm_of(grads)
        p0 = {n: s.get(n) for n in names}
        s.clip_grad_norm(share * norm)
        assert abs(s.grad_norm() - norm) <= 4 * U * norm
        for n in names:
            assert np.array_equal(s.get(n, GET_GRAD), grads[n])
        c = min(1.0, share * norm / (norm + 1e-6))
        s.optimizer_step()
        s.synchronize()
        for n in names:
            g = grads[n].astype(np.float64) * c
            m = s.get(n, GET_MOMENTUM).astype(np.float64)
            if kind == "adamw":    # m = (1 - beta1) g in the first step
                assert np.all(np.abs(m - 0.1 * g) <= 8 * U * np.abs(0.1 * g) + 1e-38), n
            else:                  # m = g + weight_decay p
                want = g + s.cfg.weight_decay * p0[n].astype(np.float64)
                assert np.all(np.abs(m - want) <= 8 * U * (np.abs(g) + np.abs(want)) + 1e-38), n
    finally:
        s.close()


@pytest.mark.parametrize("make", [gpt2, qwen2, resnet], ids=lambda f: f.__name__)
def test_a_later_pass_takes_it_back_and_one_step_uses_it_up(make):
    def momentum(clip):
        s, backward, _ = make()
        try:
            backward()
            if clip:
                s.clip_grad_norm(1e-3)
            backward()
            s.optimizer_step()
            backward()
            s.optimizer_step()
            s.synchronize()
            return {n: s.get(n) for n in s.params}
        finally:
            s.close()
    a, b = momentum(False), momentum(True)
    assert all(np.array_equal(a[n], b[n]) for n in a)


def test_accumulated_gradients_are_what_is_measured():
    s, backward, _ = gpt2()
    try:
        backward()
        s.accumulate()
        backward()
        two = {n: s.get(n, GET_GRAD) for n in s.params}
        s.accumulate()
        s.clip_grad_norm(1.0)
        want = norm_of(two)   # the same batch twice: the sum is twice one of them
        assert abs(s.grad_norm() - 2 * want) <= 8 * U * 2 * want
    finally:
        s.close()


def test_refusals():
    from sirius_b200._lib import SrtError
    s, backward, _ = gpt2()
    try:
        with pytest.raises(SrtError):
            s.grad_norm()
        backward()
        for bad in (0.0, -1.0, float("nan")):
            with pytest.raises(SrtError):
                s.clip_grad_norm(bad)
    finally:
        s.close()
    assert ops.tc_status() == 0
