"""Tensor-level wrappers over the C ABI: each takes CUDA torch tensors (used only as device
buffers) and calls one entry point on the current stream. Layouts are NHWC / KRSC."""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import ConvDesc, ConvEpilogue, IMPL_AUTO, SRT_BF16, SRT_F32, call


def _dt(t: torch.Tensor) -> int:
    if t.dtype == torch.float32:
        return SRT_F32
    if t.dtype == torch.bfloat16:
        return SRT_BF16
    raise TypeError(f"unsupported dtype {t.dtype}")


def _p(t):
    if t is None:
        return None
    assert t.is_cuda and t.is_contiguous(), "device-resident contiguous tensor required"
    return t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _check(what, shape, dtype, device, **tensors):
    """Each of `tensors` is a contiguous CUDA tensor on the current device (whose stream the call goes to), beside `device`,
    of this shape and type. None passes; a shape or type of None is not looked at."""
    for name, t in tensors.items():
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or not t.is_cuda or not t.is_contiguous():
            raise ValueError(f"{what}: {name} must be a contiguous CUDA tensor")
        if t.device != device or t.device.index != torch.cuda.current_device():
            raise ValueError(f"{what}: {name} is on {t.device}; operands are on the current device, cuda:{torch.cuda.current_device()}")
        if dtype is not None and t.dtype != dtype:
            raise TypeError(f"{what}: {name} is {t.dtype}, not {dtype}")
        if shape is not None and tuple(t.shape) != tuple(shape):
            raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, not {tuple(shape)}")


def _device(what, t):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{what}: tensors are wanted")
    return t.device


def _ep(bias, addend, addend_bits=None):
    if bias is None and addend is None:
        return None
    return C.byref(ConvEpilogue(_p(bias), _p(addend), _p(addend_bits)))


def conv_fprop(x, w, stride, pad, bias=None, addend=None, impl=IMPL_AUTO, out=None):
    N, H, W, Cin = x.shape
    K, R, S, _ = w.shape
    d = ConvDesc.make(N, H, W, Cin, K, R, S, stride, pad)
    y = out if out is not None else torch.empty((N, d.P, d.Q, K), dtype=x.dtype, device=x.device)
    call("srt_conv_fprop", C.byref(d), _dt(x), impl, _p(x), _p(w), _p(y), _ep(bias, addend), _stream())
    return y


def conv_fprop_bn_stats(x, w, stride, pad, gamma, beta, running_mean, running_var, eps=1e-5, momentum=0.1,
                        bias=None, addend=None, impl=IMPL_AUTO):
    """Convolution whose epilogue takes the BatchNorm sums of its output, then the finalize step:
    returns (y, mean, invstd, scale, shift) like conv_fprop followed by bn_stats."""
    N, H, W, Cin = x.shape
    K, R, S, _ = w.shape
    d = ConvDesc.make(N, H, W, Cin, K, R, S, stride, pad)
    if not _lib.lib().srt_conv_fprop_bn_stats_supported(C.byref(d), _dt(x), impl):
        raise RuntimeError("conv_fprop_bn_stats: this dtype/impl has no statistics epilogue")
    y = torch.empty((N, d.P, d.Q, K), dtype=x.dtype, device=x.device)
    nbytes = _lib.lib().srt_conv_fprop_bn_stats_bytes(C.byref(d))
    partial = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    slabs = C.c_int(0)
    call("srt_conv_fprop_bn_stats", C.byref(d), _dt(x), impl, _p(x), _p(w), _p(y), _ep(bias, addend), _p(partial),
         nbytes, C.byref(slabs), _stream())
    f = lambda: torch.empty(K, dtype=torch.float32, device=x.device)
    mean, invstd, scale, shift = f(), f(), f(), f()
    call("srt_bn_finalize", _p(partial), slabs.value, K, N * d.P * d.Q, _p(gamma), _p(beta), eps, momentum,
         _p(running_mean), _p(running_var), _p(mean), _p(invstd), _p(scale), _p(shift), _stream())
    return y, mean, invstd, scale, shift


def filter_transpose(w):
    K, R, S, Cin = w.shape
    d = ConvDesc.make(1, R, S, Cin, K, R, S, 1, 0)
    wt = torch.empty((Cin, R, S, K), dtype=w.dtype, device=w.device)
    call("srt_conv_filter_transpose", C.byref(d), _dt(w), _p(w), _p(wt), _stream())
    return wt


def conv_dgrad(dy, wt, x_shape, stride, pad, addend=None, impl=IMPL_AUTO, addend_bits=None):
    N, H, W, Cin = x_shape
    _, R, S, K = wt.shape
    d = ConvDesc.make(N, H, W, Cin, K, R, S, stride, pad)
    dx = torch.empty((N, H, W, Cin), dtype=dy.dtype, device=dy.device)
    call("srt_conv_dgrad", C.byref(d), _dt(dy), impl, _p(dy), _p(wt), _p(dx), _ep(None, addend, addend_bits), _stream())
    return dx


def conv_wgrad(dy, x, R, S, stride, pad, impl=IMPL_AUTO):
    N, H, W, Cin = x.shape
    K = dy.shape[-1]
    d = ConvDesc.make(N, H, W, Cin, K, R, S, stride, pad)
    nbytes = _lib.lib().srt_conv_wgrad_scratch_bytes(C.byref(d), _dt(x), impl)
    scratch = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=x.device)
    dw = torch.empty((K, R, S, Cin), dtype=torch.float32, device=x.device)
    call("srt_conv_wgrad", C.byref(d), _dt(x), impl, _p(dy), _p(x), _p(dw), _p(scratch), nbytes, _stream())
    return dw


def bn_scratch(rows, Cc, device):
    n = _lib.lib().srt_bn_scratch_bytes(rows, Cc)
    return torch.empty(n, dtype=torch.uint8, device=device), n


def bn_stats(z, gamma, beta, running_mean, running_var, eps=1e-5, momentum=0.1):
    Cc = z.shape[-1]
    rows = z.numel() // Cc
    f = lambda: torch.empty(Cc, dtype=torch.float32, device=z.device)
    mean, invstd, scale, shift = f(), f(), f(), f()
    scratch, n = bn_scratch(rows, Cc, z.device)
    call("srt_bn_stats", _dt(z), _p(z), rows, Cc, _p(gamma), _p(beta), eps, momentum, _p(running_mean),
         _p(running_var), _p(mean), _p(invstd), _p(scale), _p(shift), _p(scratch), n, _stream())
    return mean, invstd, scale, shift


def bn_apply(z, scale, shift, residual=None, relu=True):
    Cc = z.shape[-1]
    y = torch.empty_like(z)
    call("srt_bn_apply", _dt(z), _p(z), _p(residual), _p(y), z.numel() // Cc, Cc, _p(scale), _p(shift),
         int(relu), _stream())
    return y


def bn_apply_bits(z, scale, shift, residual=None):
    """bn_apply under a ReLU that also returns the mask as one bit per element (uint8 [numel / 8])."""
    Cc = z.shape[-1]
    y = torch.empty_like(z)
    bits = torch.empty(z.numel() // 8, dtype=torch.uint8, device=z.device)
    call("srt_bn_apply_bits", _dt(z), _p(z), _p(residual), _p(y), z.numel() // Cc, Cc, _p(scale), _p(shift), _p(bits), _stream())
    return y, bits


def bn_backward_bits(dy, bits, z, gamma, mean, invstd, want_dresidual=False, one_launch=False):
    Cc = z.shape[-1]
    rows = z.numel() // Cc
    dz = torch.empty_like(z)
    dres = torch.empty_like(z) if want_dresidual else None
    dgamma = torch.empty(Cc, dtype=torch.float32, device=z.device)
    dbeta = torch.empty_like(dgamma)
    scratch, n = bn_scratch(rows, Cc, z.device)
    call("srt_bn_backward_bits", _dt(z), _p(dy), _p(bits), _p(z), rows, Cc, _p(gamma), _p(mean), _p(invstd), _p(dz), _p(dres),
         _p(dgamma), _p(dbeta), _p(scratch), n, int(one_launch), _stream())
    return dz, dres, dgamma, dbeta


def bn_backward(dy, y, z, gamma, mean, invstd, relu=True, want_dresidual=False, scale=None, shift=None):
    Cc = z.shape[-1]
    rows = z.numel() // Cc
    dz = torch.empty_like(z)
    dres = torch.empty_like(z) if want_dresidual else None
    dgamma = torch.empty(Cc, dtype=torch.float32, device=z.device)
    dbeta = torch.empty_like(dgamma)
    scratch, n = bn_scratch(rows, Cc, z.device)
    call("srt_bn_backward", _dt(z), _p(dy), _p(y), _p(z), rows, Cc, _p(gamma), _p(mean), _p(invstd),
         _p(scale), _p(shift), int(relu), _p(dz), _p(dres), _p(dgamma), _p(dbeta), _p(scratch), n, _stream())
    return dz, dres, dgamma, dbeta


def bn_fused_fits(z, backward=False) -> bool:
    Cc = z.shape[-1]
    return bool(_lib.lib().srt_bn_fused_fits(_dt(z), z.numel() // Cc, Cc, int(backward)))


def bn_forward_fused(z, gamma, beta, running_mean, running_var, residual=None, relu=True, eps=1e-5, momentum=0.1):
    """Statistics + apply in one cooperative launch; returns (y, mean, invstd, scale, shift)."""
    Cc = z.shape[-1]
    f = lambda: torch.empty(Cc, dtype=torch.float32, device=z.device)
    mean, invstd, scale, shift = f(), f(), f(), f()
    y = torch.empty_like(z)
    call("srt_bn_forward_fused", _dt(z), _p(z), _p(residual), _p(y), z.numel() // Cc, Cc, _p(gamma), _p(beta), eps, momentum,
         _p(running_mean), _p(running_var), _p(mean), _p(invstd), _p(scale), _p(shift), int(relu), _stream())
    return y, mean, invstd, scale, shift


def bn_backward_fused(dy, y, z, gamma, mean, invstd, relu=True, want_dresidual=False, scale=None, shift=None):
    Cc = z.shape[-1]
    dz = torch.empty_like(z)
    dres = torch.empty_like(z) if want_dresidual else None
    dgamma = torch.empty(Cc, dtype=torch.float32, device=z.device)
    dbeta = torch.empty_like(dgamma)
    call("srt_bn_backward_fused", _dt(z), _p(dy), _p(y), _p(z), z.numel() // Cc, Cc, _p(gamma), _p(mean), _p(invstd),
         _p(scale), _p(shift), int(relu), _p(dz), _p(dres), _p(dgamma), _p(dbeta), _stream())
    return dz, dres, dgamma, dbeta


def maxpool_fwd(x):
    N, H, W, Cc = x.shape
    P, Q = (H - 1) // 2 + 1, (W - 1) // 2 + 1
    y = torch.empty((N, P, Q, Cc), dtype=x.dtype, device=x.device)
    arg = torch.empty((N, P, Q, Cc), dtype=torch.uint8, device=x.device)
    call("srt_maxpool3x3s2_fwd", _dt(x), _p(x), _p(y), _p(arg), N, H, W, Cc, _stream())
    return y, arg


def maxpool_bwd(dy, arg, x_shape):
    N, H, W, Cc = x_shape
    dx = torch.empty(x_shape, dtype=dy.dtype, device=dy.device)
    call("srt_maxpool3x3s2_bwd", _dt(dy), _p(dy), _p(arg), _p(dx), N, H, W, Cc, _stream())
    return dx


def avgpool_fwd(x):
    N, H, W, Cc = x.shape
    y = torch.empty((N, Cc), dtype=x.dtype, device=x.device)
    call("srt_avgpool_fwd", _dt(x), _p(x), _p(y), N, H * W, Cc, _stream())
    return y


def avgpool_bwd(dy, HW):
    N, Cc = dy.shape
    dx = torch.empty((N, HW, Cc), dtype=dy.dtype, device=dy.device)
    call("srt_avgpool_bwd", _dt(dy), _p(dy), _p(dx), N, HW, Cc, _stream())
    return dx


def softmax_ce(logits, labels, grad_scale):
    B, classes = logits.shape
    row_loss = torch.empty(B, dtype=torch.float32, device=logits.device)
    dlogits = torch.empty_like(logits)
    call("srt_softmax_ce", _dt(logits), _p(logits), _p(labels), B, classes, float(grad_scale),
         _p(row_loss), _p(dlogits), _stream())
    return row_loss, dlogits


def colsum(dy):
    rows, K = dy.shape
    out = torch.empty(K, dtype=torch.float32, device=dy.device)
    call("srt_colsum", _dt(dy), _p(dy), rows, K, _p(out), _stream())
    return out


def sgd_momentum(p, g, m, lr, mu, wd, first_step, p_bf16=None, clip=None):
    """`clip` as in adamw."""
    if clip is not None:
        _clip_operands(p, g, m, p_bf16, clip)
        call("srt_sgd_momentum_clipped", _p(p), _p(g), _p(m), _p(p_bf16), p.numel(), lr, mu, wd, int(first_step), _p(clip), _stream())
        return
    call("srt_sgd_momentum", _p(p), _p(g), _p(m), _p(p_bf16), p.numel(), lr, mu, wd, int(first_step), _stream())


def adamw(p, g, m, v, lr, b1, b2, eps, wd, step, p_bf16=None, clip=None):
    """`clip`: what grad_norm returned; the gradients are multiplied by its coefficient on the way in."""
    if clip is not None:
        _clip_operands(p, g, m, v, p_bf16, clip)
        call("srt_adamw_clipped", _p(p), _p(g), _p(m), _p(v), _p(p_bf16), p.numel(), lr, b1, b2, eps, wd, step, _p(clip), _stream())
        return
    call("srt_adamw", _p(p), _p(g), _p(m), _p(v), _p(p_bf16), p.numel(), lr, b1, b2, eps, wd, step, _stream())


def _clip_operands(p, *rest):
    *state, p_bf16, clip = rest
    dev = _device("clipped step", p)
    _check("clipped step", None, torch.float32, dev, p=p)
    for t in state:
        _check("clipped step", p.shape, torch.float32, dev, state=t)
    _check("clipped step", p.shape, torch.bfloat16, dev, p_bf16=p_bf16)
    _check("clipped step", (2,), torch.float32, dev, clip=clip)


def _grad_list(name, grads, max_norm):
    grads = list(grads)
    if not max_norm > 0:
        raise ValueError(f"{name}: max_norm ({max_norm}) must be positive")
    dev = grads[0].device if grads else torch.device("cuda", torch.cuda.current_device())
    dtype = grads[0].dtype if grads else torch.float32
    for g in grads:
        _check(name, None, dtype, dev, gradient=g)
    n = len(grads)
    nbytes = _lib.lib().srt_grad_norm_scratch_bytes(n)
    # the results first, the partial sums behind them
    work = torch.empty(256 + nbytes, dtype=torch.uint8, device=dev)
    clip = work[:8].view(torch.float32)
    call("srt_" + name, SRT_F32 if dtype == torch.float32 else _dt(grads[0]), n, (C.c_void_p * n)(*[g.data_ptr() for g in grads]),
         (C.c_int64 * n)(*[g.numel() for g in grads]), max_norm, clip.data_ptr(), work.data_ptr() + 256, nbytes, _stream())
    return clip


def grad_norm(grads, max_norm):
    """Norm of all gradients together (a list of tensors of one type) and the coefficient that brings it down to `max_norm`,
    min(1, max_norm / (norm + 1e-6)): a device tensor of these two, for the `clip` argument of the optimizer steps."""
    return _grad_list("grad_norm", grads, max_norm)


def clip_grad_norm(grads, max_norm):
    """grad_norm that also multiplies the gradients by the coefficient, in place (torch.nn.utils.clip_grad_norm_)."""
    return _grad_list("clip_grad_norm", grads, max_norm)


def _rows(what, x, gamma, residual):
    dev = _device(what, x)
    if x.dim() < 1 or x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"{what}: rows of float32 or bfloat16 are wanted, not {x.dtype}")
    _check(what, None, None, dev, x=x)
    _check(what, x.shape, x.dtype, dev, residual=residual)
    _check(what, x.shape[-1:], torch.float32, dev, gamma=gamma)
    return dev, x.shape[-1], x.numel() // max(x.shape[-1], 1)


def rmsnorm(x, gamma, eps=1e-6, residual=None):
    """h = x + residual, y = gamma * h / rms(h) over the last axis: returns (y, h, rstd). Without a residual h is x itself."""
    dev, Cc, rows = _rows("rmsnorm", x, gamma, residual)
    y = torch.empty_like(x)
    h = torch.empty_like(x) if residual is not None else None
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    call("srt_rmsnorm_fwd", _dt(x), _p(x), _p(residual), _p(gamma), _p(h), _p(y), _p(rstd), rows, Cc, eps, _stream())
    return y, x if h is None else h, rstd


def rmsnorm_e4m3(x, gamma, eps=1e-6, residual=None):
    """rmsnorm whose output leaves in 8 bits, q * scale of its row: returns (q, scale, h, rstd)."""
    dev, Cc, rows = _rows("rmsnorm_e4m3", x, gamma, residual)
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=dev)
    h = torch.empty_like(x) if residual is not None else None
    rstd, scale = (torch.empty(x.shape[:-1], dtype=torch.float32, device=dev) for _ in range(2))
    call("srt_rmsnorm_fwd_e4m3", _dt(x), _p(x), _p(residual), _p(gamma), _p(h), _p(q), _p(scale), _p(rstd), rows, Cc, eps, _stream())
    return q, scale, x if h is None else h, rstd


def quantize_rows_e4m3(x):
    """Rows (of weights, say) in 8 bits: (q, scale) with x close to q * scale."""
    dev, Cc, rows = _rows("quantize_rows_e4m3", x, None, None)
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=dev)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    call("srt_quantize_rows_e4m3", _dt(x), _p(x), _p(q), _p(scale), rows, Cc, _stream())
    return q, scale


def rmsnorm_backward(dy, h, gamma, rstd, dh=None):
    """Gradient of rmsnorm at the h and rstd that it returned: (dx, dgamma). dx is the gradient of x and of the residual; `dh`
    is what reaches h from elsewhere (the residual path) and is added to it."""
    dev, Cc, rows = _rows("rmsnorm_backward", h, gamma, dh)
    _check("rmsnorm_backward", h.shape, h.dtype, dev, dy=dy)
    _check("rmsnorm_backward", h.shape[:-1], torch.float32, dev, rstd=rstd)
    dx = torch.empty_like(h)
    dgamma = torch.empty(Cc, dtype=torch.float32, device=dev)
    nbytes = _lib.lib().srt_rmsnorm_bwd_scratch_bytes(Cc)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    call("srt_rmsnorm_bwd", _dt(h), _p(dy), _p(h), _p(gamma), _p(rstd), _p(dh), _p(dx), _p(dgamma), rows, Cc, _p(scratch), nbytes, _stream())
    return dx, dgamma


def _ffn(what, x, w_gate_up, w_down, dtype):
    dev = _device(what, x)
    _check(what, None, dtype, dev, x=x, w_gate_up=w_gate_up)
    _check(what, None, torch.bfloat16, dev, w_down=w_down)
    if x.dim() != 2 or w_gate_up.dim() != 2 or w_down.dim() != 2 or w_gate_up.shape[0] != 2 * w_down.shape[1]:
        raise ValueError(f"{what}: x [tokens, width], w_gate_up [2 hidden, width] and w_down [width, hidden] are wanted, not "
                         f"{tuple(x.shape)}, {tuple(w_gate_up.shape)} and {tuple(w_down.shape)}")
    (tokens, width), hidden = x.shape, w_down.shape[1]
    if w_gate_up.shape[1] != width or w_down.shape[0] != width:
        raise ValueError(f"{what}: x has {width} columns, w_gate_up {w_gate_up.shape[1]} and w_down {w_down.shape[0]} rows")
    return dev, _lib.GatedFfnDesc(tokens, width, hidden)


def gated_ffn(x, w_gate_up, w_down, residual=None):
    """residual + (silu(x Wg^T) * (x Wu^T)) Wd^T with w_gate_up = Wg over Wu; bf16."""
    dev, d = _ffn("gated_ffn", x, w_gate_up, w_down, torch.bfloat16)
    _check("gated_ffn", x.shape, torch.bfloat16, dev, residual=residual)
    nbytes = _lib.lib().srt_gated_ffn_fwd_scratch_bytes(C.byref(d))
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    y = torch.empty_like(x)
    call("srt_gated_ffn_fwd", C.byref(d), _p(x), _p(w_gate_up), _p(w_down), _p(residual), _p(y), _p(scratch), nbytes, _stream())
    return y


def gated_ffn_e4m3(x, x_scale, w_gate_up, w_scale, w_down, residual=None):
    """gated_ffn on 8-bit rows: x * x_scale of its row (rmsnorm_e4m3) and w_gate_up * w_scale of its row (quantize_rows_e4m3)."""
    dev, d = _ffn("gated_ffn_e4m3", x, w_gate_up, w_down, torch.float8_e4m3fn)
    _check("gated_ffn_e4m3", (d.tokens,), torch.float32, dev, x_scale=x_scale)
    _check("gated_ffn_e4m3", (2 * d.hidden,), torch.float32, dev, w_scale=w_scale)
    _check("gated_ffn_e4m3", x.shape, torch.bfloat16, dev, residual=residual)
    nbytes = _lib.lib().srt_gated_ffn_fwd_scratch_bytes(C.byref(d))
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    y = torch.empty(x.shape, dtype=torch.bfloat16, device=dev)
    call("srt_gated_ffn_fwd_e4m3", C.byref(d), _p(x), _p(x_scale), _p(w_gate_up), _p(w_scale), _p(w_down), _p(residual), _p(y), _p(scratch),
         nbytes, _stream())
    return y


def gated_ffn_backward(dy, x, w_gate_up, w_down, grad_dtype=torch.bfloat16):
    """Gradients of gated_ffn at x, which is all that forward has to keep: (dx, dw_gate_up, dw_down), the weights' in
    `grad_dtype` (bfloat16, or float32 for an optimizer that accumulates there). The residual's gradient is dy itself."""
    dev, d = _ffn("gated_ffn_backward", x, w_gate_up, w_down, torch.bfloat16)
    _check("gated_ffn_backward", x.shape, torch.bfloat16, dev, dy=dy)
    if grad_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"gated_ffn_backward: gradients in bfloat16 or float32, not {grad_dtype}")
    g = SRT_F32 if grad_dtype == torch.float32 else SRT_BF16
    dx, dw_gate_up, dw_down = torch.empty_like(x), torch.empty_like(w_gate_up, dtype=grad_dtype), torch.empty_like(w_down, dtype=grad_dtype)
    nbytes = _lib.lib().srt_gated_ffn_bwd_scratch_bytes(C.byref(d), g)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    call("srt_gated_ffn_bwd", C.byref(d), _p(dy), _p(x), _p(w_gate_up), _p(w_down), g, _p(dx), _p(dw_gate_up), _p(dw_down), _p(scratch),
         nbytes, _stream())
    return dx, dw_gate_up, dw_down


def grad_accumulate(acc, g):
    call("srt_grad_accumulate", _p(acc), _p(g), acc.numel(), _stream())


def nchw_to_nhwc(src, dtype, Cpad):
    N, Cc, H, W = src.shape
    dst = torch.empty((N, H, W, Cpad), dtype=dtype, device=src.device)
    call("srt_nchw_to_nhwc", SRT_F32 if dtype == torch.float32 else SRT_BF16, _p(src), _p(dst), N, Cc, H, W,
         Cpad, _stream())
    return dst


def tc_status() -> int:
    s = C.c_int(0)
    call("srt_tc_status", C.byref(s))
    return s.value
