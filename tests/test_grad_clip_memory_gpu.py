"""The first clip_grad_norm of an executor takes no device memory: what it needs was laid out with the step, so it neither waits in the
allocator nor fails in the middle of an update while inference holds the rest of the device."""
import ctypes as C

import pytest
import torch
from test_grad_clip_executors_gpu import gpt2, qwen2, resnet, swin

pytestmark = pytest.mark.gpu


def free_memory():
    """Free device memory: the driver gives small requests parts of pieces of 2 MB, so one shows here when it opens a new piece."""
    torch.cuda.synchronize()
    return torch.cuda.mem_get_info()[0]


@pytest.mark.parametrize("make", [gpt2, qwen2, swin, resnet], ids=lambda f: f.__name__)
def test_the_first_call_takes_no_memory(make):
    s, backward, _ = make()
    runtime = C.CDLL("libcudart.so.12")
    filler = []
    try:
        backward()
        s.optimizer_step()   # whatever the launches of a step load is loaded
        backward()
        other, again, _ = make()
        again()
        other.clip_grad_norm(1.0)
        other.optimizer_step()
        other.synchronize()
        other.close()
        # close the gaps of pieces that are open already: small requests until one opens a new piece, which is given back
        for _ in range(4096):
            before, p = free_memory(), C.c_void_p()
            assert runtime.cudaMalloc(C.byref(p), C.c_size_t(8448)) == 0
            if free_memory() < before:   # the pieces that were open are full
                assert runtime.cudaFree(p) == 0
                break
            filler.append(p)
        else:
            pytest.fail("no request opened a new piece")
        before = free_memory()
        s.clip_grad_norm(1.0)
        s.optimizer_step()
        s.synchronize()
        assert free_memory() == before
    finally:
        for p in filler:
            runtime.cudaFree(p)
        s.close()
