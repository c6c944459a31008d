"""Qwen2 step whose MLPs keep no projections (recompute_mlp): the tests of the step itself, against the same oracle and fixtures,
and what the mode saves."""
import json
import pathlib

import numpy as np
import pytest

from oracle import qwen2_oracle as O
from sirius_b200 import ops
from sirius_b200.qwen2_step import GET_GRAD, Qwen2Step

pytestmark = pytest.mark.gpu
TINY = dict(n_layer=2, n_head=4, n_kv_head=2, hidden=128, intermediate=256, vocab=500)


@pytest.mark.parametrize("case", ["qwen2_tiny", "qwen2_05b_b4_s2048"])
def test_against_the_committed_golden_fixture(case):
    from parity import check_gradient_digests, check_update_digests
    doc = json.loads((pathlib.Path(__file__).parent / "golden" / f"{case}.json").read_text())
    cfg, B, S, steps, ref = doc["config"], doc["batch"], doc["seq"], doc["steps"], doc["fp32"]
    model = O.build_model(**cfg, seed=doc["seed"])
    batches = O.make_tokens(B, S, cfg["vocab"], steps, seed=doc["seed"])
    step = Qwen2Step(**cfg, max_batch=B, seq=S, recompute_mlp=True)
    init = O.state_arrays(model)
    step.load_state_dict(init)
    del model
    losses = []
    for i, ids in enumerate(batches):
        step.upload_tokens(ids)
        step.forward_backward()
        if i == 0:
            assert abs(step.loss() - ref["loss0"]) < 2e-2 * abs(ref["loss0"])
            check_gradient_digests(lambda n: step.get(n, GET_GRAD), ref["grad0"], what=case)
        step.optimizer_step()
        losses.append(step.loss())
    for a, b in zip(losses, ref["losses"]):
        assert abs(a - b) < 2e-2 * abs(b), (losses, ref["losses"])
    check_update_digests(step.get, init, ref["delta"], ref["final"], doc["optimizer"]["lr"], steps, what=case)
    assert ops.tc_status() == 0
    step.close()


def grads_of(step, ids):
    step.upload_tokens(ids)
    step.forward_backward()
    return step.loss(), {n: step.get(n, GET_GRAD) for n in step.params}


def test_repeats_bit_for_bit_and_can_be_switched():
    B, S = 2, 128
    state = O.state_arrays(O.build_model(**TINY, seed=0))
    ids = O.make_tokens(B, S, TINY["vocab"], 1)[0]
    step = Qwen2Step(**TINY, max_batch=B, seq=S)
    step.load_state_dict(state)
    plain = grads_of(step, ids)
    step.recompute_mlp()
    a, b = grads_of(step, ids), grads_of(step, ids)
    assert a[0] == b[0] and all(np.array_equal(a[1][n], b[1][n]) for n in a[1])
    assert abs(a[0] - plain[0]) < 1e-2 * abs(plain[0])
    step.recompute_mlp(False)
    c = grads_of(step, ids)
    assert c[0] == plain[0] and all(np.array_equal(c[1][n], plain[1][n]) for n in plain[1])
    step.close()
    assert ops.tc_status() == 0


def test_keeps_six_bytes_less_per_token_layer_and_channel():
    cfg = dict(n_layer=12, n_head=4, n_kv_head=2, hidden=256, intermediate=2048, vocab=500)
    a = Qwen2Step(**cfg, max_batch=4, seq=512)
    before = a.memory_bytes()
    a.recompute_mlp()
    saved = before - a.memory_bytes()
    tokens = 4 * 512
    # the layers' own, less the scratch that takes their place once (the activation, twice it, the slots of shared tiles)
    assert saved >= 6 * tokens * 2048 * 12 - 40 * 2 ** 20, saved
    assert saved <= 6 * tokens * 2048 * 12 + 6 * tokens * 2048
    a.close()


def test_shrunk_and_regained_batches():
    state = O.state_arrays(O.build_model(**TINY, seed=0))
    ids = O.make_tokens(4, 128, TINY["vocab"], 1)[0]
    step = Qwen2Step(**TINY, max_batch=4, seq=128, recompute_mlp=True)
    step.load_state_dict(state)
    whole = grads_of(step, ids)
    step.shrink_activations(2)
    small = grads_of(step, ids[:2])
    again = grads_of(step, ids)
    assert again[0] == whole[0] and all(np.array_equal(again[1][n], whole[1][n]) for n in whole[1])
    fresh = Qwen2Step(**TINY, max_batch=2, seq=128, recompute_mlp=True)
    fresh.load_state_dict(state)
    two = grads_of(fresh, ids[:2])
    assert two[0] == small[0] and all(np.array_equal(two[1][n], small[1][n]) for n in two[1])
    step.close()
    fresh.close()


def test_memory_line_of_the_adjuster():
    """As for the other executors: what the trainer registers as model "qwen_recompute" has a line of its own, half as steep."""
    import ctypes as C
    import gc

    import torch

    from sirius_b200 import mem_model
    from sirius_b200._lib import call
    gc.collect()
    torch.cuda.empty_cache()
    got = mem_model.measure(("qwen_recompute",))["qwen_recompute"]
    base, slope = C.c_double(), C.c_double()
    call("srt_adjuster_model_mem_param_measured", b"qwen_recompute", C.byref(base), C.byref(slope))
    for batch, mb in zip(got["batches"], got["device_mb"]):
        assert abs(base.value + slope.value * batch - mb) <= 0.1 * mb, (got, base.value, slope.value)
    assert abs(slope.value - got["slope_mb"]) <= 0.1 * got["slope_mb"], (got, slope.value)


@pytest.mark.parametrize("recompute", [False, True])
def test_clipped_steps_on_a_partition_of_the_device(recompute):
    """The step and its clipping while training has a part of the SMs: kernels are cut for that width, the work is the same."""
    import ctypes as C

    from sirius_b200._lib import call
    full = (1 << 64) - 1
    B, S = 2, 128
    state = O.state_arrays(O.build_model(**TINY, seed=0))
    ids = O.make_tokens(B, S, TINY["vocab"], 1)[0]

    def run(mask):
        step = Qwen2Step(**TINY, max_batch=B, seq=S, recompute_mlp=recompute)
        try:
            step.load_state_dict(state)
            if mask is not None:
                step.follow_sm_mask(True)
                call("srt_set_sm_mask", (C.c_uint64 * 3)(*mask))
            loss, grads = grads_of(step, ids)
            step.clip_grad_norm(0.5)
            return loss, grads, step.grad_norm(), step.current_sms()
        finally:
            call("srt_set_sm_mask", (C.c_uint64 * 3)(full, full, full))
            step.close()
    whole, part = run(None), run((full, 0, 0))
    assert part[3] <= 64 < whole[3]
    assert abs(part[0] - whole[0]) <= 1e-3 * abs(whole[0]) and abs(part[2] - whole[2]) <= 2e-2 * whole[2]
    top = max(float(np.linalg.norm(g)) for g in whole[1].values())
    for n, g in whole[1].items():
        # sums cut elsewhere round elsewhere: the same bound as against the oracle
        assert np.linalg.norm(part[1][n] - g) <= 5e-2 * np.linalg.norm(g) + 1e-3 * top, n
    assert ops.tc_status() == 0
