"""The gradients of a list live until the call on them has ended, whatever other threads do to the list meanwhile.

A copy of the native front end is bound to a stand-in for the library whose entry point launches nothing: it tells that it was
reached and waits. The interpreter's lock is given up there, so this thread can empty the list and look at what is still held."""
import ctypes as C
import importlib.util
import shutil
import subprocess
import threading
import time

import pytest
import torch

from sirius_b200 import _build, _lib

pytestmark = pytest.mark.gpu

STAND_IN = r"""
#include <stddef.h>
#include <time.h>
volatile int entered = 0, leave = 0;
const char* srt_last_error(void) { return ""; }
size_t srt_grad_norm_scratch_bytes(int n) { return 8192; }
static int wait_here(void) {
  struct timespec t = {0, 1000000};
  entered = 1;
  for (int i = 0; i < 20000 && !leave; ++i) nanosleep(&t, 0);
  return leave ? 0 : 1;
}
int srt_grad_norm() { return wait_here(); }
int srt_clip_grad_norm() { return wait_here(); }
#define NOTHING(name) int name() { return 1; }
NOTHING(srt_rmsnorm_fwd) NOTHING(srt_rmsnorm_fwd_e4m3) NOTHING(srt_quantize_rows_e4m3) NOTHING(srt_rmsnorm_bwd_scratch_bytes)
NOTHING(srt_rmsnorm_bwd) NOTHING(srt_gated_ffn_fwd_scratch_bytes) NOTHING(srt_gated_ffn_fwd) NOTHING(srt_gated_ffn_fwd_e4m3)
NOTHING(srt_gated_ffn_bwd_scratch_bytes) NOTHING(srt_gated_ffn_bwd) NOTHING(srt_adamw_clipped) NOTHING(srt_sgd_momentum_clipped)
"""


@pytest.fixture
def front(tmp_path):
    (tmp_path / "stand_in.c").write_text(STAND_IN)
    lib = tmp_path / "libstand_in.so"
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", str(tmp_path / "stand_in.c"), "-o", str(lib)], check=True)
    copy = tmp_path / "_ops_native.so"
    shutil.copy(_build.BINDING, copy)
    spec = importlib.util.spec_from_file_location("_ops_native", copy)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.bind(str(lib), _lib.SrtError, torch.OutOfMemoryError)
    return module, C.CDLL(str(lib))


@pytest.mark.parametrize("in_place", [False, True])
def test_a_list_that_another_thread_empties(front, in_place):
    module, lib = front
    entered, leave = C.c_int.in_dll(lib, "entered"), C.c_int.in_dll(lib, "leave")
    torch.cuda.synchronize()
    start = torch.cuda.memory_allocated()
    grads = [torch.zeros(1 << 20, device="cuda") for _ in range(3)]
    held = torch.cuda.memory_allocated() - start
    assert held >= 3 << 22
    out = []

    def run():
        try:
            out.append(module.grad_norm(grads, 1.0, in_place))
        except Exception as e:
            out.append(e)
    t = threading.Thread(target=run)
    t.start()
    try:
        t0 = time.time()
        while not entered.value:
            assert time.time() - t0 < 15
            time.sleep(0.001)
        grads.clear()
        during = torch.cuda.memory_allocated() - start
    finally:
        leave.value = 1
        t.join(30)
    assert not t.is_alive() and isinstance(out[0], torch.Tensor), out
    assert during >= held, "the gradients were freed while the call ran on them"
    out.clear()
    assert torch.cuda.memory_allocated() == start
