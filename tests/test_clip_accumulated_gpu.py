"""Clipping through the trainer's loop on the executors: the update of a global batch of two micro-batches is the one that the
calls written by hand make, bit for bit, and it is clipped; a request that accumulating would take back is an error."""
import contextlib

import numpy as np
import pytest

from sirius_b200 import ops
from sirius_b200 import torch_col as tc
from sirius_b200.torch_col import dynamic_batch as db
from test_grad_clip_executors_gpu import gpt2, qwen2, resnet, swin

pytestmark = pytest.mark.gpu


class Batch(dict):
    def should_update_param(self):
        return self["do_step"]


@pytest.fixture
def mgr(monkeypatch):
    class Ctrl:
        @contextlib.contextmanager
        def steps_no_interrupt(self):
            yield
    monkeypatch.setattr(db, "get_colocate_ctrl", lambda: Ctrl())
    monkeypatch.setattr(db.MicroBatchManager, "_micro_batch_manager", None)
    yield db.MicroBatchManager(None, enable_grad_accumulate=True, checkpoint_micro_batch=True)
    db.MicroBatchManager._micro_batch_manager = None
    tc.EventManager.reset()


@pytest.mark.parametrize("make", [gpt2, qwen2, resnet], ids=lambda f: f.__name__)
def test_the_loop_clips_the_sum_of_the_micro_batches(make, mgr):
    def by_hand(max_norm):
        s, backward, _ = make()
        try:
            for _ in range(2):
                backward()
                s.accumulate()
            if max_norm:
                s.clip_grad_norm(max_norm)
                assert s.clip_pending
            s.optimizer_step()
            s.synchronize()
            assert not s.clip_pending
            return {n: s.get(n) for n in s.params}, s.grad_norm() if max_norm else None
        finally:
            s.close()
    _, norm = by_hand(1.0)
    want, plain = by_hand(norm / 4)[0], by_hand(None)[0]
    assert any(not np.array_equal(want[n], plain[n]) for n in want)
    for max_norm, expected in ((norm / 4, want), (None, plain)):
        s, backward, _ = make()
        acc = tc.GradAccumulator(s)
        try:
            for k in range(2):
                backward()
                mgr.optimizer_step(Batch(do_step=k == 1), s, grad_accumulator=acc, max_norm=max_norm)
            s.synchronize()
            if max_norm:
                assert s.grad_norm() == norm
            assert all(np.array_equal(s.get(n), expected[n]) for n in expected)
        finally:
            s.close()
    assert ops.tc_status() == 0


@pytest.mark.parametrize("make", [gpt2, resnet], ids=lambda f: f.__name__)
def test_a_request_that_accumulating_would_take_back(make, mgr):
    s, backward, _ = make()
    try:
        backward()
        s.clip_grad_norm(1e-3)
        with pytest.raises(RuntimeError, match="max_norm"):
            mgr.optimizer_step(Batch(do_step=True), s, grad_accumulator=tc.GradAccumulator(s))
        assert s.clip_pending
    finally:
        s.close()


@pytest.mark.parametrize("make", [gpt2, qwen2, swin, resnet], ids=lambda f: f.__name__)
def test_what_takes_a_request_back(make):
    s, backward, _ = make()
    try:
        assert not s.clip_pending
        backward()
        s.clip_grad_norm(1.0)
        assert s.clip_pending
        backward()
        assert not s.clip_pending
        if hasattr(s, "accumulate"):
            s.clip_grad_norm(1.0)
            s.accumulate()
            assert not s.clip_pending
        s.clip_grad_norm(1.0)
        s.optimizer_step()
        assert not s.clip_pending
    finally:
        s.close()
