"""Tensor-level wrappers over the C ABI: each takes CUDA torch tensors (used only as device
buffers) and calls one entry point on the current stream. Layouts are NHWC / KRSC."""
from __future__ import annotations

import ctypes as C
from array import array

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


_current_device = torch.cuda.current_device
_raw_stream = torch._C._cuda_getCurrentRawStream   # the handle without the Stream object around it, which takes 3 us to make


def _stream():
    return _raw_stream(_current_device())


def _wrong(what, name, t, shape, dtype, dev):
    """The error that _check's operand deserves."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous CUDA tensor")
    if t.get_device() != dev:
        raise ValueError(f"{what}: {name} is on {t.device}; operands are on the current device, cuda:{dev}")
    if dtype is not None and t.dtype is not dtype:
        raise TypeError(f"{what}: {name} is {t.dtype}, not {dtype}")
    raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, not {tuple(shape)}")


def _check(what, name, t, shape, dtype, dev):
    """Address of a contiguous CUDA tensor of this shape and type on the current device `dev` (whose stream the call goes to).
    None gives None; a shape or type of None is not looked at."""
    if t is None:
        return None
    if (not isinstance(t, torch.Tensor) or t.get_device() != dev or not t.is_contiguous() or (dtype is not None and t.dtype is not dtype)
            or (shape is not None and t.shape != shape)):
        _wrong(what, name, t, shape, dtype, dev)
    return t.data_ptr()


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
        pp, gp, mp, _, bp, cp, st = _clip_operands("sgd_momentum", p, g, m, None, p_bf16, clip)
        call("srt_sgd_momentum_clipped", pp, gp, mp, bp, p.numel(), lr, mu, wd, int(first_step), cp, st)
        return
    call("srt_sgd_momentum", _p(p), _p(g), _p(m), _p(p_bf16), p.numel(), lr, mu, wd, int(first_step), _stream())


def adamw(p, g, m, v, lr, b1, b2, eps, wd, step, p_bf16=None, clip=None):
    """`clip`: what grad_norm returned; the gradients are multiplied by its coefficient on the way in."""
    if clip is not None:
        pp, gp, mp, vp, bp, cp, st = _clip_operands("adamw", p, g, m, v, p_bf16, clip)
        call("srt_adamw_clipped", pp, gp, mp, vp, bp, p.numel(), lr, b1, b2, eps, wd, step, cp, st)
        return
    call("srt_adamw", _p(p), _p(g), _p(m), _p(v), _p(p_bf16), p.numel(), lr, b1, b2, eps, wd, step, _stream())


def _clip_operands(what, p, g, m, v, p_bf16, clip):
    dev, f32 = _current_device(), torch.float32
    pp = _check(what, "p", p, None, f32, dev)
    shape = p.shape
    return (pp, _check(what, "g", g, shape, f32, dev), _check(what, "m", m, shape, f32, dev), _check(what, "v", v, shape, f32, dev),
            _check(what, "p_bf16", p_bf16, shape, torch.bfloat16, dev), _check(what, "clip", clip, (2,), f32, dev), _raw_stream(dev))


def _grad_list(name, grads, max_norm):
    if not max_norm > 0:
        raise ValueError(f"{name}: max_norm ({max_norm}) must be positive")
    dev = _current_device()
    if not isinstance(grads, (list, tuple)):
        grads = list(grads)
    n = len(grads)
    dtype = grads[0].dtype if n else torch.float32
    for g in grads:
        if g.get_device() != dev or g.dtype is not dtype or not g.is_contiguous():
            _wrong(name, "a gradient", g, None, dtype, dev)
    kind = _dt(grads[0]) if n else SRT_F32
    # addresses and counts behind one another, read by the call before it returns
    words = array("q", [g.data_ptr() for g in grads])
    words.extend([g.numel() for g in grads])
    at = words.buffer_info()[0]
    nbytes = _lib.lib().srt_grad_norm_scratch_bytes(n)
    # the results first, the partial sums behind them
    work = torch.empty(64 + nbytes // 4, dtype=torch.float32, device="cuda")
    base = work.data_ptr()
    call("srt_" + name, kind, n, at, at + 8 * n, max_norm, base, base + 256, nbytes, _raw_stream(dev))
    return work[:2]


def grad_norm(grads, max_norm):
    """Norm of all gradients together (a list of tensors of one type) and the coefficient that brings it down to `max_norm`,
    min(1, max_norm / (norm + 1e-6)): a device tensor of these two, for the `clip` argument of the optimizer steps."""
    return _grad_list("grad_norm", grads, max_norm)


def clip_grad_norm(grads, max_norm):
    """grad_norm that also multiplies the gradients by the coefficient, in place (torch.nn.utils.clip_grad_norm_)."""
    return _grad_list("clip_grad_norm", grads, max_norm)


def _row_type(what, x):
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        raise ValueError(f"{what}: rows in a CUDA tensor are wanted")
    if x.dtype is torch.bfloat16:
        return SRT_BF16
    if x.dtype is torch.float32:
        return SRT_F32
    raise TypeError(f"{what}: rows of float32 or bfloat16 are wanted, not {x.dtype}")


def rmsnorm(x, gamma, eps=1e-6, residual=None):
    """h = x + residual, y = gamma * h / rms(h) over the last axis: returns (y, h, rstd). Without a residual h is x itself."""
    kind, dev = _row_type("rmsnorm", x), _current_device()
    shape = x.shape
    xp = _check("rmsnorm", "x", x, None, None, dev)
    rp = _check("rmsnorm", "residual", residual, shape, x.dtype, dev)
    gp = _check("rmsnorm", "gamma", gamma, shape[-1:], torch.float32, dev)
    y = torch.empty_like(x)
    h = x if residual is None else torch.empty_like(x)
    rstd = gamma.new_empty(shape[:-1])
    call("srt_rmsnorm_fwd", kind, xp, rp, gp, None if residual is None else h.data_ptr(), y.data_ptr(), rstd.data_ptr(), rstd.numel(),
         shape[-1], eps, _raw_stream(dev))
    return y, h, rstd


def rmsnorm_e4m3(x, gamma, eps=1e-6, residual=None):
    """rmsnorm whose output leaves in 8 bits, q * scale of its row: returns (q, scale, h, rstd)."""
    kind, dev = _row_type("rmsnorm_e4m3", x), _current_device()
    shape = x.shape
    xp = _check("rmsnorm_e4m3", "x", x, None, None, dev)
    rp = _check("rmsnorm_e4m3", "residual", residual, shape, x.dtype, dev)
    gp = _check("rmsnorm_e4m3", "gamma", gamma, shape[-1:], torch.float32, dev)
    q = torch.empty_like(x, dtype=torch.float8_e4m3fn)
    h = x if residual is None else torch.empty_like(x)
    rstd, scale = gamma.new_empty(shape[:-1]), gamma.new_empty(shape[:-1])
    call("srt_rmsnorm_fwd_e4m3", kind, xp, rp, gp, None if residual is None else h.data_ptr(), q.data_ptr(), scale.data_ptr(), rstd.data_ptr(),
         rstd.numel(), shape[-1], eps, _raw_stream(dev))
    return q, scale, h, rstd


def quantize_rows_e4m3(x):
    """Rows (of weights, say) in 8 bits: (q, scale) with x close to q * scale."""
    kind, dev = _row_type("quantize_rows_e4m3", x), _current_device()
    xp = _check("quantize_rows_e4m3", "x", x, None, None, dev)
    q = torch.empty_like(x, dtype=torch.float8_e4m3fn)
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    call("srt_quantize_rows_e4m3", kind, xp, q.data_ptr(), scale.data_ptr(), scale.numel(), x.shape[-1], _raw_stream(dev))
    return q, scale


def rmsnorm_backward(dy, h, gamma, rstd, dh=None):
    """Gradient of rmsnorm at the h and rstd that it returned: (dx, dgamma). dx is the gradient of x and of the residual; `dh`
    is what reaches h from elsewhere (the residual path) and is added to it."""
    what = "rmsnorm_backward"
    kind, dev = _row_type(what, h), _current_device()
    shape, dtype = h.shape, h.dtype
    hp = _check(what, "h", h, None, None, dev)
    dyp, dhp = _check(what, "dy", dy, shape, dtype, dev), _check(what, "dh", dh, shape, dtype, dev)
    gp, rp = _check(what, "gamma", gamma, shape[-1:], torch.float32, dev), _check(what, "rstd", rstd, shape[:-1], torch.float32, dev)
    dx, dgamma = torch.empty_like(h), torch.empty_like(gamma)
    nbytes = _lib.lib().srt_rmsnorm_bwd_scratch_bytes(shape[-1])
    scratch = gamma.new_empty(nbytes // 4)
    call("srt_rmsnorm_bwd", kind, dyp, hp, gp, rp, dhp, dx.data_ptr(), dgamma.data_ptr(), rstd.numel(), shape[-1], scratch.data_ptr(), nbytes,
         _raw_stream(dev))
    return dx, dgamma


def _ffn(what, x, w_gate_up, w_down, dtype, dev):
    if not all(isinstance(t, torch.Tensor) and t.dim() == 2 for t in (x, w_gate_up, w_down)) or w_gate_up.shape[0] != 2 * w_down.shape[1]:
        raise ValueError(f"{what}: x [tokens, width], w_gate_up [2 hidden, width] and w_down [width, hidden] are wanted")
    tokens, width = x.shape
    hidden = w_down.shape[1]
    d = _lib.GatedFfnDesc(tokens, width, hidden)
    return (d, _check(what, "x", x, None, dtype, dev), _check(what, "w_gate_up", w_gate_up, (2 * hidden, width), dtype, dev),
            _check(what, "w_down", w_down, (width, hidden), torch.bfloat16, dev))


def gated_ffn(x, w_gate_up, w_down, residual=None):
    """residual + (silu(x Wg^T) * (x Wu^T)) Wd^T with w_gate_up = Wg over Wu; bf16."""
    dev = _current_device()
    d, xp, gp, wp = _ffn("gated_ffn", x, w_gate_up, w_down, torch.bfloat16, dev)
    rp = _check("gated_ffn", "residual", residual, x.shape, torch.bfloat16, dev)
    ref = C.byref(d)
    nbytes = _lib.lib().srt_gated_ffn_fwd_scratch_bytes(ref)
    scratch, y = x.new_empty(nbytes // 2), torch.empty_like(x)
    call("srt_gated_ffn_fwd", ref, xp, gp, wp, rp, y.data_ptr(), scratch.data_ptr(), nbytes, _raw_stream(dev))
    return y


def gated_ffn_e4m3(x, x_scale, w_gate_up, w_scale, w_down, residual=None):
    """gated_ffn on 8-bit rows: x * x_scale of its row (rmsnorm_e4m3) and w_gate_up * w_scale of its row (quantize_rows_e4m3)."""
    what, dev = "gated_ffn_e4m3", _current_device()
    d, xp, gp, wp = _ffn(what, x, w_gate_up, w_down, torch.float8_e4m3fn, dev)
    xs = _check(what, "x_scale", x_scale, (d.tokens,), torch.float32, dev)
    ws = _check(what, "w_scale", w_scale, (2 * d.hidden,), torch.float32, dev)
    rp = _check(what, "residual", residual, x.shape, torch.bfloat16, dev)
    ref = C.byref(d)
    nbytes = _lib.lib().srt_gated_ffn_fwd_scratch_bytes(ref)
    scratch, y = w_down.new_empty(nbytes // 2), w_down.new_empty(x.shape)
    call("srt_gated_ffn_fwd_e4m3", ref, xp, xs, gp, ws, wp, rp, y.data_ptr(), scratch.data_ptr(), nbytes, _raw_stream(dev))
    return y


def gated_ffn_backward(dy, x, w_gate_up, w_down, grad_dtype=torch.bfloat16):
    """Gradients of gated_ffn at x, which is all that forward has to keep: (dx, dw_gate_up, dw_down), the weights' in
    `grad_dtype` (bfloat16, or float32 for an optimizer that accumulates there). The residual's gradient is dy itself."""
    what, dev = "gated_ffn_backward", _current_device()
    d, xp, gp, wp = _ffn(what, x, w_gate_up, w_down, torch.bfloat16, dev)
    dyp = _check(what, "dy", dy, x.shape, torch.bfloat16, dev)
    if grad_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{what}: gradients in bfloat16 or float32, not {grad_dtype}")
    g = SRT_F32 if grad_dtype is torch.float32 else SRT_BF16
    dx, dw_gate_up, dw_down = torch.empty_like(x), torch.empty_like(w_gate_up, dtype=grad_dtype), torch.empty_like(w_down, dtype=grad_dtype)
    ref = C.byref(d)
    nbytes = _lib.lib().srt_gated_ffn_bwd_scratch_bytes(ref, g)
    scratch = x.new_empty(nbytes // 2)
    call("srt_gated_ffn_bwd", ref, dyp, xp, gp, wp, g, dx.data_ptr(), dw_gate_up.data_ptr(), dw_down.data_ptr(), scratch.data_ptr(), nbytes,
         _raw_stream(dev))
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
