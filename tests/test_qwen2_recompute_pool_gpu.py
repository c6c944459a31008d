"""recompute_mlp on a page pool: a pool that holds the mode's own activations is enough to create the step, and switching the mode on
hands the pages that it saves back to the pool."""
from contextlib import ExitStack

import numpy as np
import pytest

from oracle import qwen2_oracle as O
from sirius_b200 import ops
from sirius_b200._lib import SrtError
from sirius_b200.pool import PagePool
from sirius_b200.qwen2_step import GET_GRAD, Qwen2Step

pytestmark = pytest.mark.gpu
CFG = dict(n_layer=8, n_head=4, n_kv_head=2, hidden=256, intermediate=2048, vocab=500)
B, S = 4, 512


def sizes():
    """Bytes of the activations: with the projections kept, and with recompute_mlp."""
    s = Qwen2Step(**CFG, max_batch=B, seq=S)
    try:
        plain = s.memory_bytes()
        s.recompute_mlp()
        recompute = s.memory_bytes()
        s.release_activations()
        return plain - s.memory_bytes(), recompute - s.memory_bytes()
    finally:
        s.close()


def gradients(step, state, ids):
    step.load_state_dict(state)
    step.upload_tokens(ids)
    step.forward_backward()
    return step.loss(), {n: step.get(n, GET_GRAD) for n in step.params}


def test_a_pool_that_holds_the_modes_own_activations_is_enough():
    plain, recompute = sizes()
    assert plain - recompute > 128 << 20
    state = O.state_arrays(O.build_model(**CFG, seed=0))
    ids = O.make_tokens(B, S, CFG["vocab"], 1)[0]
    alone = Qwen2Step(**CFG, max_batch=B, seq=S, recompute_mlp=True)
    want = gradients(alone, state, ids)
    alone.close()
    with ExitStack() as ends:   # the steps before their pool, whatever fails
        pool = PagePool((recompute + (plain - recompute) / 2) / 2 ** 30, page_mb=2)
        ends.callback(pool.close)
        with pytest.raises(SrtError):
            Qwen2Step(**CFG, max_batch=B, seq=S, pool=pool.handle)
        assert pool.stat("train_usage") == 0
        step = Qwen2Step(**CFG, max_batch=B, seq=S, pool=pool.handle, recompute_mlp=True)
        ends.callback(step.close)
        got = gradients(step, state, ids)
        assert got[0] == want[0] and all(np.array_equal(got[1][n], want[1][n]) for n in want[1])
    assert ops.tc_status() == 0

def test_switching_hands_the_saved_pages_back():
    plain, recompute = sizes()
    with ExitStack() as ends:
        pool = PagePool((plain + (256 << 20)) / 2 ** 30, page_mb=2)
        ends.callback(pool.close)
        step = Qwen2Step(**CFG, max_batch=B, seq=S, pool=pool.handle)
        ends.callback(step.close)
        before = pool.stat("free_pages")
        step.recompute_mlp()
        gained = (pool.stat("free_pages") - before) * pool.stat("page_nbytes")
        # whole pages of 2 MB, of which every block may share its first and its last with a neighbour
        assert gained >= 0.9 * (plain - recompute), (gained, plain - recompute)
        step.recompute_mlp(False)
        assert pool.stat("free_pages") <= before + 8
