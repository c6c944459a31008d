"""GradAccumulator (pytorch/torch_col/accumulate.py:7-49): keeps the gradient of the global batch while
micro-batches come and go, so a killed micro-batch only loses its own work.

Two back ends with the same three methods: a sirius_b200 step object (the accumulation and the
optimizer run as fused kernels over its flat buffers) or a torch.nn.Module (the reference's code path,
used on CPU ranks in the tests)."""
from __future__ import annotations

from collections import defaultdict


def clip_module_grads(params, max_norm, optimizer=None, scaler=None):
    """Clipping of a torch module's gradients, which a loss scaler has to unscale first."""
    import torch
    if scaler is not None:
        scaler.unscale_(optimizer)
    torch.nn.utils.clip_grad_norm_(params, max_norm)


class GradAccumulator:
    def __init__(self, model, exchange=None):
        """exchange: a sirius_b200.ddp.GradExchange for data-parallel training with a step object. The ranks of a
        job may run different numbers of micro-batches per global batch, so what they exchange is the accumulated
        gradient, once, right before the update (DDP's no_sync on every micro-batch but the last,
        pytorch/torch_col/dynamic_batch.py:155-167)."""
        self._step = model if hasattr(model, 'optimizer_step') and hasattr(model, 'accumulate') else None
        self._exchange = exchange
        if exchange is not None and self._step is None:
            raise ValueError("a GradExchange works on a step object; torch modules bring their own all-reduce")
        if self._step is None:
            import torch
            self.param_list = [p for p in model.parameters() if p.requires_grad]
            self.param_grads = defaultdict(dict)
            for p in self.param_list:
                self.param_grads[p]['global'] = torch.zeros_like(p)
                self.param_grads[p]['local'] = None

    def accumulate(self):
        if self._step is not None:
            if getattr(self._step, 'clip_pending', False):   # accumulating takes it back, and the update would go unclipped
                raise RuntimeError("clip_grad_norm before accumulate is lost: pass max_norm to GradAccumulator.step or "
                                   "MicroBatchManager.optimizer_step")
            return self._step.accumulate()
        for p in self.param_list:
            self.param_grads[p]['global'] += p.grad
            p.grad.zero_()

    def step(self, optimizer=None, scaler=None, do_zero_grad=True, max_norm=None):
        """max_norm: the accumulated gradient of the global batch, summed over the ranks, is scaled by
        min(1, max_norm / its norm) on its way into the update."""
        if self._step is not None:
            if self._exchange is not None:
                self._exchange.allreduce(self._step, accumulated=True)   # sum over ranks, on the library's NCCL stream
            if max_norm is not None:
                self._step.clip_grad_norm(max_norm)
            return self._step.optimizer_step()  # uses and then clears the accumulated gradient
        for p in self.param_list:
            self.param_grads[p]['local'] = p.grad
            p.grad = self.param_grads[p]['global']
        if max_norm is not None:
            clip_module_grads(self.param_list, max_norm, optimizer, scaler)
        if scaler is not None:
            scaler.step(optimizer)
            scaler.update()
        else:
            optimizer.step()
        for p in self.param_list:
            p.grad = self.param_grads[p]['local']
        if do_zero_grad:
            self.zero_grad()

    def zero_grad(self):
        if self._step is None:
            for p in self.param_list:
                self.param_grads[p]['global'].zero_()
