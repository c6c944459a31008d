"""Clipping in the trainer's own loop: MicroBatchManager.optimizer_step and GradAccumulator.step take max_norm, the norm is that of
the global batch's accumulated gradient (behind the exchange between ranks), and a clip_grad_norm that accumulating would take
back is an error instead of an unclipped update."""
import contextlib

import pytest
import torch

from sirius_b200 import torch_col as tc
from sirius_b200.torch_col import dynamic_batch as db
from sirius_b200.torch_col.accumulate import GradAccumulator


class Step:
    """The calls that a step object gets, in order, and the rule of the executors: accumulating takes a coefficient back."""

    def __init__(self):
        self.calls, self.clip_pending = [], False

    def accumulate(self):
        self.calls.append("accumulate")
        self.clip_pending = False

    def clip_grad_norm(self, max_norm):
        self.calls.append(("clip", max_norm))
        self.clip_pending = True

    def optimizer_step(self):
        self.calls.append("clipped update" if self.clip_pending else "update")
        self.clip_pending = False


class Exchange:
    def allreduce(self, step, accumulated=False):
        step.calls.append("exchange" if accumulated else "exchange of one micro-batch")


class Batch(dict):
    def __init__(self, last):
        super().__init__(do_step=last)

    def should_update_param(self):
        return self["do_step"]


@pytest.fixture
def manager(monkeypatch):
    class Ctrl:
        @contextlib.contextmanager
        def steps_no_interrupt(self):
            yield
    monkeypatch.setattr(db, "get_colocate_ctrl", lambda: Ctrl())
    monkeypatch.setattr(db.MicroBatchManager, "_micro_batch_manager", None)

    def make(**kw):
        db.MicroBatchManager._micro_batch_manager = None
        return db.MicroBatchManager(None, **kw)
    yield make
    db.MicroBatchManager._micro_batch_manager = None
    tc.EventManager.reset()


def test_the_sum_of_the_micro_batches_is_clipped_behind_the_exchange(manager):
    mgr, step = manager(enable_grad_accumulate=True, checkpoint_micro_batch=True), Step()
    acc = GradAccumulator(step, exchange=Exchange())
    for last in (False, False, True, True):
        mgr.optimizer_step(Batch(last), step, grad_accumulator=acc, max_norm=0.5)
    update = ["exchange", ("clip", 0.5), "clipped update"]
    assert step.calls == ["accumulate"] * 3 + update + ["accumulate"] + update


def test_without_a_bound_nothing_is_measured(manager):
    mgr, step = manager(enable_grad_accumulate=True, checkpoint_micro_batch=True), Step()
    acc = GradAccumulator(step)
    mgr.optimizer_step(Batch(True), step, grad_accumulator=acc)
    assert step.calls == ["accumulate", "update"]


def test_a_step_object_without_an_accumulator(manager):
    mgr, step = manager(), Step()
    mgr.optimizer_step(Batch(True), step, max_norm=2.0)
    mgr.optimizer_step(Batch(True), step)
    assert step.calls == [("clip", 2.0), "clipped update", "update"]


def test_a_request_that_accumulating_would_take_back_is_an_error(manager):
    mgr, step = manager(enable_grad_accumulate=True, checkpoint_micro_batch=True), Step()
    acc = GradAccumulator(step)
    step.clip_grad_norm(1.0)
    with pytest.raises(RuntimeError, match="max_norm"):
        mgr.optimizer_step(Batch(True), step, grad_accumulator=acc)
    assert step.calls == [("clip", 1.0)]


@pytest.mark.parametrize("bad", [0.0, -1.0, float("nan")])
def test_bounds_are_refused_before_anything_is_accumulated(manager, bad):
    mgr, step = manager(enable_grad_accumulate=True, checkpoint_micro_batch=True), Step()
    with pytest.raises(ValueError, match="max_norm"):
        mgr.optimizer_step(Batch(True), step, grad_accumulator=GradAccumulator(step), max_norm=bad)
    assert step.calls == []


def pair(seed=0):
    torch.manual_seed(seed)
    a = torch.nn.Sequential(torch.nn.Linear(6, 5), torch.nn.Tanh(), torch.nn.Linear(5, 3)).double()
    b = torch.nn.Sequential(torch.nn.Linear(6, 5), torch.nn.Tanh(), torch.nn.Linear(5, 3)).double()
    b.load_state_dict(a.state_dict())
    x = torch.randn(3, 4, 6, dtype=torch.float64)
    return a, b, x


@pytest.mark.parametrize("share", [0.2, 5.0])
@pytest.mark.parametrize("scaled", [False, True])
def test_a_torch_module(manager, share, scaled):
    """Three micro-batches against one batch of all: the same clipped update, with and without a loss scaler (a power of two, so
    that unscaling is exact). The sums meet in another order, 2^-50 of values below one."""
    a, b, x = pair()
    (b(x.reshape(12, 6)).square().sum()).backward()
    norm = float(torch.nn.utils.clip_grad_norm_(b.parameters(), float("inf")))
    torch.nn.utils.clip_grad_norm_(b.parameters(), share * norm)
    torch.optim.SGD(b.parameters(), 0.125).step()

    mgr = manager(enable_grad_accumulate=True, checkpoint_micro_batch=True)
    opt, acc = torch.optim.SGD(a.parameters(), 0.125), GradAccumulator(a)
    scaler = torch.amp.GradScaler("cpu", init_scale=2.0 ** 10) if scaled else None
    for k in range(3):
        loss = a(x[k]).square().sum()
        (scaler.scale(loss) if scaled else loss).backward()
        mgr.optimizer_step(Batch(k == 2), opt, scaler, acc, max_norm=share * norm)
    for p, q in zip(a.parameters(), b.parameters()):
        assert (p - q).abs().max() <= 2.0 ** -40


@pytest.mark.parametrize("scaled", [False, True])
def test_a_torch_module_without_an_accumulator(manager, scaled):
    a, b, x = pair(1)
    (b(x[0]).square().sum()).backward()
    torch.nn.utils.clip_grad_norm_(b.parameters(), 0.01)
    torch.optim.SGD(b.parameters(), 0.125).step()
    opt = torch.optim.SGD(a.parameters(), 0.125)
    scaler = torch.amp.GradScaler("cpu", init_scale=2.0 ** 10) if scaled else None
    loss = a(x[0]).square().sum()
    (scaler.scale(loss) if scaled else loss).backward()
    manager().optimizer_step(Batch(True), opt, scaler, max_norm=0.01)
    for p, q in zip(a.parameters(), b.parameters()):
        assert (p - q).abs().max() <= 2.0 ** -40
