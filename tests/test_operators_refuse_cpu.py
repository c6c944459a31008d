"""What the operators of the feed-forward half and of the optimizer step refuse, at the tensor level and at the C entry points;
nothing here reaches a device."""
import ctypes as C

import pytest
import torch

from sirius_b200 import _lib, ops
from sirius_b200._lib import GatedFfnDesc, SRT_BF16, SRT_F32

BF = torch.bfloat16
x, wgu, wd, gamma = torch.zeros(4, 16, dtype=BF), torch.zeros(16, 16, dtype=BF), torch.zeros(16, 8, dtype=BF), torch.zeros(16)


@pytest.mark.parametrize("f", [
    lambda: ops.rmsnorm(x, gamma), lambda: ops.rmsnorm_e4m3(x, gamma), lambda: ops.quantize_rows_e4m3(x),
    lambda: ops.rmsnorm_backward(x, x, gamma, torch.zeros(4)), lambda: ops.gated_ffn(x, wgu, wd),
    lambda: ops.gated_ffn_e4m3(x, gamma, wgu, gamma, wd), lambda: ops.gated_ffn_backward(x, x, wgu, wd),
    lambda: ops.grad_norm([gamma], 1.0), lambda: ops.clip_grad_norm([gamma], 1.0),
    lambda: ops.adamw(gamma, gamma, gamma, gamma, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, clip=gamma[:2]),
    lambda: ops.sgd_momentum(gamma, gamma, gamma, 1e-3, 0.9, 0.0, False, clip=gamma[:2])])
def test_host_tensors_are_refused(f):
    with pytest.raises(ValueError, match="must be a contiguous CUDA tensor"):
        f()


@pytest.mark.parametrize("f", [lambda: ops.rmsnorm(None, gamma), lambda: ops.rmsnorm(3.0, gamma), lambda: ops.gated_ffn([1], wgu, wd),
                               lambda: ops.grad_norm([None], 1.0)])
def test_other_objects_are_refused(f):
    with pytest.raises(ValueError, match="must be a contiguous CUDA tensor"):
        f()


def test_bounds_of_the_norm_and_gradient_types():
    for bad in (0.0, -1.0, float("nan")):
        for f in (ops.grad_norm, ops.clip_grad_norm):
            with pytest.raises(ValueError, match="max_norm"):
                f([gamma], bad)
    with pytest.raises(TypeError):
        ops.grad_norm(gamma.sum, 1.0)
    with pytest.raises(TypeError):
        ops.grad_norm([gamma], "x")
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        ops.gated_ffn_backward(x, x, wgu, wd, grad_dtype=torch.float16)


def status(name, *args):
    rc = getattr(_lib.lib(), name)(*args)
    return rc, _lib.lib().srt_last_error().decode()


P = 1 << 20  # an address that no refused call looks at


@pytest.mark.parametrize("rows,c,dtype,word", [(4, 12, SRT_F32, "multiple of 8"), (4, 0, SRT_F32, "multiple of 8"), (4, -8, SRT_F32, "multiple of 8"),
                                               (4, 16392, SRT_BF16, "longer"), (4, 8200, SRT_F32, "longer"), (-1, 8, SRT_F32, "not negative"),
                                               (1 << 31, 8, SRT_F32, "2^31"), (4, 8, 7, "dtype")])
def test_rows_that_the_norms_refuse(rows, c, dtype, word):
    for name, args in (("srt_rmsnorm_fwd", (dtype, P, None, P, None, P, None, rows, c, 1e-6, None)),
                       ("srt_rmsnorm_fwd_e4m3", (dtype, P, None, P, None, P, P, None, rows, c, 1e-6, None)),
                       ("srt_quantize_rows_e4m3", (dtype, P, P, P, rows, c, None)),
                       ("srt_rmsnorm_bwd", (dtype, P, P, P, P, None, P, P, rows, c, P, 1 << 40, None))):
        rc, text = status(name, *args)
        assert rc == 1 and word in text, (name, rc, text)


def test_pointers_that_the_norms_refuse():
    for name, args in (("srt_rmsnorm_fwd", (SRT_F32, P + 4, None, P, None, P, None, 4, 8, 1e-6, None)),
                       ("srt_rmsnorm_fwd", (SRT_F32, P, P + 8, P, None, P, None, 4, 8, 1e-6, None)),
                       ("srt_rmsnorm_fwd_e4m3", (SRT_F32, P, None, P, None, P + 8, P, None, 4, 8, 1e-6, None)),
                       ("srt_quantize_rows_e4m3", (SRT_F32, P, P + 1, P, 4, 8, None)),
                       ("srt_rmsnorm_bwd", (SRT_F32, P, P, P, P, None, P + 2, P, 4, 8, P, 1 << 40, None))):
        rc, text = status(name, *args)
        assert rc == 1 and "aligned" in text, (name, rc, text)
    for name, args in (("srt_rmsnorm_fwd", (SRT_F32, None, None, P, None, P, None, 4, 8, 1e-6, None)),
                       ("srt_rmsnorm_fwd", (SRT_F32, P, None, None, None, P, None, 4, 8, 1e-6, None)),
                       ("srt_rmsnorm_fwd_e4m3", (SRT_F32, P, None, P, None, P, None, None, 4, 8, 1e-6, None)),
                       ("srt_rmsnorm_bwd", (SRT_F32, P, P, P, None, None, P, P, 4, 8, P, 1 << 40, None)),
                       ("srt_rmsnorm_bwd", (SRT_F32, P, P, P, P, None, P, None, 4, 8, P, 1 << 40, None))):
        rc, text = status(name, *args)
        assert rc == 1 and "null" in text, (name, rc, text)
    rc, text = status("srt_rmsnorm_bwd", SRT_F32, P, P, P, P, None, P, P, 4, 8, P, _lib.lib().srt_rmsnorm_bwd_scratch_bytes(8) - 1, None)
    assert rc == 1 and "scratch" in text


BAD_SIZES = [((-1, 8, 8), "out of range"), ((4, 0, 8), "out of range"), ((4, 8, 0), "out of range"), ((4, 12, 8), "multiple"), ((4, 8, 12), "multiple"),
             ((1 << 20, 16, 1024), "2^31"), ((1 << 16, 1 << 15, 8), "2^31"), ((4, 1 << 16, 1 << 14), "2^31")]


@pytest.mark.parametrize("sizes,word", BAD_SIZES)
def test_sizes_that_the_block_refuses(sizes, word):
    d = C.byref(GatedFfnDesc(*sizes))
    for name, args in (("srt_gated_ffn_fwd", (d, P, P, P, None, P, P, 1 << 50, None)),
                       ("srt_gated_ffn_fwd_e4m3", (d, P, P, P, P, P, None, P, P, 1 << 50, None)),
                       ("srt_gated_ffn_bwd", (d, P, P, P, P, SRT_F32, P, P, P, P, 1 << 50, None))):
        rc, text = status(name, *args)
        assert rc == 1 and word in text, (name, rc, text)
    assert _lib.lib().srt_gated_ffn_fwd_scratch_bytes(d) == 0 and _lib.lib().srt_gated_ffn_bwd_scratch_bytes(d, SRT_F32) == 0


def test_operands_that_the_block_refuses():
    d = C.byref(GatedFfnDesc(4, 24, 16))
    cases = [("srt_gated_ffn_fwd", (None, P, P, P, None, P, P, 1 << 50, None), "null"),
             ("srt_gated_ffn_fwd", (d, P, None, P, None, P, P, 1 << 50, None), "null"),
             ("srt_gated_ffn_fwd", (d, P + 8, P, P, None, P, P, 1 << 50, None), "aligned"),
             ("srt_gated_ffn_fwd", (d, P, P, P, P + 2, P, P, 1 << 50, None), "aligned"),
             ("srt_gated_ffn_fwd", (d, P, P, P, None, P, P, 64, None), "scratch"),
             ("srt_gated_ffn_fwd", (d, P, P, P, None, P, None, 1 << 50, None), "scratch"),
             ("srt_gated_ffn_fwd_e4m3", (d, P, P, P, P, P, None, P, P, 1 << 50, None), "multiple of 16"),
             ("srt_gated_ffn_bwd", (d, P, P, P, None, SRT_F32, P, P, P, P, 1 << 50, None), "null"),
             ("srt_gated_ffn_bwd", (d, P, P, P, P, 5, P, P, P, P, 1 << 50, None), "gradient type"),
             ("srt_gated_ffn_bwd", (d, P, P, P, P, SRT_F32, P, P + 4, P, P, 1 << 50, None), "aligned"),
             ("srt_gated_ffn_bwd", (d, P, P, P, P, SRT_F32, P, P, P, P, 128, None), "scratch")]
    for name, args, word in cases:
        rc, text = status(name, *args)
        assert rc == 1 and word in text, (name, rc, text)
    d16 = C.byref(GatedFfnDesc(4, 32, 16))
    rc, text = status("srt_gated_ffn_fwd_e4m3", d16, P, None, P, P, P, None, P, P, 1 << 50, None)
    assert rc == 1 and "null" in text


def test_lists_that_the_gradient_norm_refuses():
    ptr, n = (C.c_void_p * 2)(P, P + 64), (C.c_int64 * 2)(4, 4)
    need = _lib.lib().srt_grad_norm_scratch_bytes(2)
    for name in ("srt_grad_norm", "srt_clip_grad_norm"):
        for args, word in (((9, 2, ptr, n, 1.0, P, P, need, None), "dtype"), ((SRT_F32, -1, ptr, n, 1.0, P, P, need, None), "null"),
                           ((SRT_F32, 2, None, n, 1.0, P, P, need, None), "null"), ((SRT_F32, 2, ptr, n, 1.0, None, P, need, None), "null"),
                           ((SRT_F32, 2, ptr, n, 0.0, P, P, need, None), "positive"), ((SRT_F32, 2, ptr, n, float("nan"), P, P, need, None), "positive"),
                           ((SRT_F32, 2, ptr, n, 1.0, P, P, need - 1, None), "scratch"), ((SRT_F32, 2, ptr, n, 1.0, P, P + 4, need, None), "scratch"),
                           ((SRT_F32, 2, (C.c_void_p * 2)(P, None), n, 1.0, P, P, need, None), "tensor 1"),
                           ((SRT_F32, 2, ptr, (C.c_int64 * 2)(4, -4), 1.0, P, P, need, None), "tensor 1"),
                           ((SRT_F32, 2, (C.c_void_p * 2)(P, P + 2), n, 1.0, P, P, need, None), "aligned"),
                           ((SRT_BF16, 2, (C.c_void_p * 2)(P + 1, P), n, 1.0, P, P, need, None), "aligned")):
            rc, text = status(name, *args)
            assert rc == 1 and word in text, (name, rc, text)


def test_clipped_steps_refuse():
    for args in ((P, P, P, P, None, 4, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, None, None), (None, P, P, P, None, 4, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, P, None),
                 (P, P, P, P, None, -4, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, P, None), (P, P, P, P, None, 4, 1e-3, 0.9, 0.99, 1e-8, 0.0, 0, P, None)):
        assert status("srt_adamw_clipped", *args)[0] == 1
    assert status("srt_sgd_momentum_clipped", P, P, P, None, 4, 0.1, 0.9, 0.0, 1, None, None)[0] == 1


def test_workspaces_are_sized_on_the_host():
    lib = _lib.lib()
    assert lib.srt_grad_norm_scratch_bytes(0) == lib.srt_grad_norm_scratch_bytes(1) > 0
    assert lib.srt_grad_norm_scratch_bytes(1025) > lib.srt_grad_norm_scratch_bytes(1024)
    d = C.byref(GatedFfnDesc(100, 64, 128))
    assert lib.srt_gated_ffn_fwd_scratch_bytes(d) >= 100 * 128 * 2
    assert lib.srt_gated_ffn_bwd_scratch_bytes(d, SRT_F32) >= 100 * 128 * 6


@pytest.mark.parametrize("c", [1 << 28, 1 << 29, 1 << 30, (1 << 31) - 8])
def test_rows_whose_bytes_pass_32_bits(c):
    for dtype in (SRT_F32, SRT_BF16):
        rc, text = status("srt_rmsnorm_fwd", dtype, P, None, P, None, P, None, 1, c, 1e-6, None)
        assert rc == 1 and "longer" in text


def test_pointers_between_two_elements():
    for name, args in (("srt_rmsnorm_fwd", (SRT_F32, P, None, P + 2, None, P, None, 4, 8, 1e-6, None)),
                       ("srt_rmsnorm_fwd_e4m3", (SRT_F32, P, None, P, None, P, P + 1, None, 4, 8, 1e-6, None)),
                       ("srt_rmsnorm_bwd", (SRT_F32, P, P, P, P, None, P, P + 2, 4, 8, P, 1 << 40, None)),
                       ("srt_gated_ffn_fwd_e4m3", (C.byref(GatedFfnDesc(4, 32, 16)), P, P + 2, P, P, P, None, P, P, 1 << 50, None)),
                       ("srt_grad_norm", (SRT_F32, 0, None, None, 1.0, P + 2, P, 1 << 40, None)),
                       ("srt_adamw_clipped", (P + 2, P, P, P, None, 4, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, P, None)),
                       ("srt_adamw_clipped", (P, P, P, P, P + 1, 4, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, P, None)),
                       ("srt_sgd_momentum_clipped", (P, P, P, None, 4, 0.1, 0.9, 0.0, 1, P + 1, None))):
        rc, text = status(name, *args)
        assert rc == 1 and "aligned" in text, (name, rc, text)
