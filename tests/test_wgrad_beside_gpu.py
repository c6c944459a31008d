"""Filter gradients that the transformer executors queue on their second stream take the kernel without CTA pairs, whatever the
process-wide switch says: the gradients are those of a process with the switch off, bit for bit. The sizes are such that pairs would
cut the reduction elsewhere (of 960 x 320 over 4096 tokens they make 8 parts, single CTAs 11; of 576 x 192 over 12544 they make 22 and
28), so their sums would differ in the last bits, which is shown on the kernel alone, one launch on one stream."""
import numpy as np
import pytest
import torch

from sirius_b200 import _lib, ops
from sirius_b200.gpt2_step import GET_GRAD, Gpt2Step
from sirius_b200.qwen2_step import Qwen2Step
from sirius_b200.swin_step import SwinStep

pytestmark = pytest.mark.gpu


def gpt2():
    s = Gpt2Step(n_layer=2, n_head=5, d_model=320, vocab=512, ctx=1024, max_batch=4, seq=1024)
    rng = np.random.default_rng(0)
    s.load_state_dict({n: rng.normal(0, 0.02, sh).astype(np.float32) for n, (_, sh) in s.params.items()})
    s.upload_tokens(rng.integers(0, 512, (4, 1024)))
    return s


def qwen2():
    s = Qwen2Step(n_layer=2, n_head=5, n_kv_head=1, hidden=320, intermediate=640, vocab=512, max_batch=4, seq=1024)
    rng = np.random.default_rng(1)
    s.load_state_dict({n: (1 if "norm" in n else 0) + rng.normal(0, 0.02, sh).astype(np.float32) for n, (_, sh) in s.params.items()})
    s.upload_tokens(rng.integers(0, 512, (4, 1024)))
    return s


def swin():
    s = SwinStep(image=224, patch=4, embed=96, depths=(1, 1, 1, 1), heads=(3, 6, 12, 24), window=7, num_classes=40, max_batch=16)
    rng = np.random.default_rng(2)
    s.load_state_dict({n: (1 if "norm" in n and n.endswith("weight") else 0) + rng.normal(0, 0.02, sh).astype(np.float32) for n, (_, sh) in s.params.items()})
    g = torch.Generator().manual_seed(2)
    s.upload_batch(torch.randn(16, 3, 224, 224, generator=g), torch.randint(0, 40, (16,), generator=g))
    return s


def with_switch(on, f):
    before = _lib.lib().srt_conv_wgrad_pairs(on)
    try:
        return f()
    finally:
        _lib.lib().srt_conv_wgrad_pairs(before)


@pytest.mark.parametrize("make", [gpt2, qwen2, swin], ids=lambda f: f.__name__)
def test_the_switch_does_not_reach_the_second_stream(make):
    s = make()
    names = [n for n in s.params if "running" not in n]

    def grads():
        s.forward_backward()
        return {n: s.get(n, GET_GRAD) for n in names}
    try:
        on, off = with_switch(1, grads), with_switch(0, grads)
        assert all(np.array_equal(on[n], off[n]) for n in names)
        assert ops.tc_status() == 0
    finally:
        s.close()


@pytest.mark.parametrize("filters,columns,tokens", [(960, 320, 4096), (576, 192, 12544)])
def test_the_kernels_differ_in_the_last_bits(filters, columns, tokens):
    g = torch.Generator(device="cuda").manual_seed(3)
    dy = torch.randn(tokens, 1, 1, filters, device="cuda", generator=g).bfloat16()
    x = torch.randn(tokens, 1, 1, columns, device="cuda", generator=g).bfloat16()
    call = lambda: ops.conv_wgrad(dy, x, 1, 1, 1, 0)
    on, off = with_switch(1, call), with_switch(0, call)
    want = dy.view(tokens, filters).double().T @ x.view(tokens, columns).double()
    terms = dy.view(tokens, filters).double().abs().T @ x.view(tokens, columns).double().abs()
    for got in (on, off):
        assert ((got.view(filters, columns).double() - want).abs() <= tokens * 2.0 ** -23 * terms).all()
    assert not torch.equal(on, off) and ops.tc_status() == 0
