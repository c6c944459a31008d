"""Gated feed-forward block (bf16, and e4m3 operands) against its definition in 64 bits, at sizes around the tiles.

Tolerances, per element: every rounding to bf16 is off by at most 2^-8 of the value; a reduction of K products in fp32 by at
most K 2^-23 of the sum of their magnitudes; the exponential and the quotient of the sigmoid by 2^-18. What a rounding does to
a result goes through the absolute values of the following product."""
import ctypes as C

import pytest
import torch

from sirius_b200 import _lib, ops

pytestmark = pytest.mark.gpu
BF, E8 = torch.bfloat16, torch.float8_e4m3fn
H = 2.0 ** -8       # half a step of bf16
S = 2.0 ** -18      # sigmoid in fp32

# tokens, width, hidden: one token; tiles not filled and filled to the last row; widths below and beyond a k-block; hidden
# channels below a tile, odd multiples of eight, several tiles; pairs of CTAs from about a thousand tokens on
SIZES = [(1, 896, 4864), (1, 8, 8), (2, 64, 24), (3, 1544, 1032), (4, 40, 4104), (5, 72, 264), (7, 72, 40), (8, 128, 136), (24, 1040, 2008), (127, 64, 64), (128, 96, 512), (129, 136, 1032),
         (255, 200, 72), (333, 896, 1064), (1000, 264, 1096), (1024, 896, 2432), (2049, 136, 4872), (4100, 64, 1160)]


def make(t, c, f, seed=0, std=0.7):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * t + c + f)
    n = lambda *s: torch.randn(s, device="cuda", generator=g)
    return {"x": n(t, c).to(BF), "wgu": (n(2 * f, c) * (std * c ** -0.5)).to(BF), "wd": (n(c, f) * (std * f ** -0.5)).to(BF),
            "res": n(t, c).to(BF), "dy": n(t, c).to(BF)}


def reference(x, wgu, wd, res=None, dy=None, dx_terms=True):
    """Values and error bounds in 64 bits: y, and with dy the three gradients."""
    x, wgu, wd = x.double(), wgu.double(), wd.double()
    (t, c), f = x.shape, wd.shape[1]
    acc = lambda k: k * 2.0 ** -23
    g, u = (x @ wgu.T).split(f, 1)
    eg, eu = (acc(c) * (x.abs() @ wgu.abs().T)).split(f, 1)
    s = torch.sigmoid(g)
    silu = g * s
    act = silu * u
    e_act = 1.1 * u.abs() * eg + silu.abs() * eu + S * act.abs()
    if dy is None:
        y = act @ wd.T + (0 if res is None else res.double())
        ey = H * y.abs() + (H * (act.abs() + e_act) + e_act) @ wd.abs().T + acc(f) * (act.abs() @ wd.abs().T)
        return y, ey * 1.01
    dy = dy.double()
    da = dy @ wd
    ea = acc(c) * (dy.abs() @ wd.abs())
    ds = s * (1 + g * (1 - s))
    dg, du = da * u * ds, da * silu
    e_dg = 1.1 * u.abs() * ea + 1.1 * da.abs() * eu + 0.5 * da.abs() * u.abs() * eg + S * 1.1 * (da * u).abs()
    e_du = silu.abs() * ea + 1.1 * da.abs() * eg + S * du.abs()
    dgu, e_dgu = torch.cat([dg, du], 1), torch.cat([e_dg, e_du], 1)
    e_dgu = e_dgu + H * (dgu.abs() + e_dgu)
    e_ar = e_act + H * (act.abs() + e_act)
    dx, dw, dd = dgu @ wgu, dgu.T @ x, dy.T @ act
    ex = e_dgu @ wgu.abs() + acc(2 * f) * (dgu.abs() @ wgu.abs())
    ew = e_dgu.T @ x.abs() + acc(t) * (dgu.abs().T @ x.abs())
    ed = dy.abs().T @ e_ar + acc(t) * (dy.abs().T @ act.abs())
    return (dx, dw, dd), (ex, ew, ed)


def close(got, want, tol, what):
    d = (got.double() - want).abs()
    assert torch.isfinite(got.double()).all(), what
    worst = (d - tol).max()
    assert (d <= tol + 1e-30).all(), f"{what}: {int((d > tol).sum())} of {d.numel()} beyond the bound, by up to {float(worst):.3g}"


@pytest.mark.parametrize("t,c,f", SIZES)
@pytest.mark.parametrize("residual", [True, False])
def test_forward(t, c, f, residual):
    s = make(t, c, f)
    res = s["res"] if residual else None
    y = ops.gated_ffn(s["x"], s["wgu"], s["wd"], residual=res)
    assert ops.tc_status() == 0
    close(y, *reference(s["x"], s["wgu"], s["wd"], res), "y")
    assert torch.equal(y, ops.gated_ffn(s["x"], s["wgu"], s["wd"], residual=res))


@pytest.mark.parametrize("t,c,f", SIZES)
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_backward(t, c, f, dtype):
    s = make(t, c, f)
    got = ops.gated_ffn_backward(s["dy"], s["x"], s["wgu"], s["wd"], grad_dtype=dtype)
    assert ops.tc_status() == 0
    want, tol = reference(s["x"], s["wgu"], s["wd"], dy=s["dy"])
    for a, b, e, r, what in zip(got, want, tol, (H, H if dtype == BF else 2.0 ** -23, H if dtype == BF else 2.0 ** -23), ("dx", "dw_gate_up", "dw_down")):
        close(a, b, (e + r * (b.abs() + e)) * 1.01, what)
    assert got[1].dtype == dtype and got[2].dtype == dtype
    for a, b in zip(got, ops.gated_ffn_backward(s["dy"], s["x"], s["wgu"], s["wd"], grad_dtype=dtype)):
        assert torch.equal(a, b)


def test_backward_against_differences():
    """The directional derivative of sum(dy * y) along x and both weights, by central differences of the 64-bit definition."""
    t, c, f = 70, 136, 264
    s = make(t, c, f)
    got = ops.gated_ffn_backward(s["dy"], s["x"], s["wgu"], s["wd"], grad_dtype=torch.float32)
    _, tol = reference(s["x"], s["wgu"], s["wd"], dy=s["dy"])
    base = [s["x"].double(), s["wgu"].double(), s["wd"].double()]

    def loss(x, wgu, wd):
        g, u = (x @ wgu.T).split(f, 1)
        return ((g * torch.sigmoid(g) * u) @ wd.T * s["dy"].double()).sum()
    gen = torch.Generator(device="cuda").manual_seed(5)
    for k in range(3):
        d = torch.randn(base[k].shape, device="cuda", dtype=torch.float64, generator=gen)
        h = 1e-5
        plus, minus = list(base), list(base)
        plus[k], minus[k] = base[k] + h * d, base[k] - h * d
        slope = (loss(*plus) - loss(*minus)) / (2 * h)
        bound = ((tol[k] + H * got[k].double().abs()) * d.abs()).sum() + 1e-6 * slope.abs()   # the difference itself is off by h^2
        assert (got[k].double() * d).sum().sub(slope).abs() <= bound


@pytest.mark.parametrize("t,c,f", [(1, 4096, 1016), (1, 16, 8), (2, 1040, 520), (3, 32, 72), (4, 528, 1000), (5, 528, 1000), (9, 144, 40), (24, 1040, 2008), (130, 272, 520), (333, 896, 1064), (2049, 144, 4872)])
def test_e4m3(t, c, f):
    s = make(t, c, f)
    xq, xs = ops.quantize_rows_e4m3(s["x"])
    wq, ws = ops.quantize_rows_e4m3(s["wgu"])
    y = ops.gated_ffn_e4m3(xq, xs, wq, ws, s["wd"], residual=s["res"])
    assert ops.tc_status() == 0
    close(y, *reference(xq.double() * xs.double()[:, None], wq.double() * ws.double()[:, None], s["wd"], s["res"]), "y")


@pytest.mark.parametrize("t,c,f", [(130, 72, 136), (1100, 72, 1096)])
def test_a_bad_token_stays_alone(t, c, f):
    s = make(t, c, f)
    want = ops.gated_ffn(s["x"], s["wgu"], s["wd"])
    dwant = ops.gated_ffn_backward(s["dy"], s["x"], s["wgu"], s["wd"])[0]
    bad = torch.tensor([3, t - 1], device="cuda")
    x = s["x"].clone()
    x[3, 5], x[t - 1, 0] = float("nan"), float("inf")
    y = ops.gated_ffn(x, s["wgu"], s["wd"])
    dx = ops.gated_ffn_backward(s["dy"], x, s["wgu"], s["wd"])[0]
    good = torch.ones(t, dtype=torch.bool, device="cuda")
    good[bad] = False
    assert torch.equal(y[good], want[good]) and torch.equal(dx[good], dwant[good])
    assert y[bad].isnan().any(1).all()


def test_large_projections_saturate_the_gate():
    """Projections of several hundred: the exponential over- and underflows, the gate is 0 or 1, nothing becomes NaN."""
    s = make(64, 64, 72, std=300.0)
    close(ops.gated_ffn(s["x"], s["wgu"], s["wd"]), *reference(s["x"], s["wgu"], s["wd"]), "y")
    got = ops.gated_ffn_backward(s["dy"], s["x"], s["wgu"], s["wd"], grad_dtype=torch.float32)
    assert all(torch.isfinite(g.float()).all() for g in got)


def test_no_tokens():
    s = make(8, 64, 24)
    e = s["x"][:0]
    assert ops.gated_ffn(e, s["wgu"], s["wd"]).shape == (0, 64)
    dx, dw, dd = ops.gated_ffn_backward(e, e, s["wgu"], s["wd"])
    assert dx.shape == (0, 64) and not dw.any() and not dd.any() and dw.shape == s["wgu"].shape and dd.shape == s["wd"].shape


@pytest.mark.parametrize("t,c,f", [(9, 72, 40), (700, 136, 1032), (1100, 264, 2056)])
def test_rows_beyond_the_outputs_stay(t, c, f):
    """y and the gradients as slices of larger buffers: the rows behind them are left as they were."""
    s = make(t, c, f)
    d = _lib.GatedFfnDesc(t, c, f)
    st = torch.cuda.current_stream().cuda_stream
    y = torch.full((t + 3, c), 7.0, device="cuda", dtype=BF)
    n = _lib.lib().srt_gated_ffn_fwd_scratch_bytes(C.byref(d))
    scratch = torch.full((n + 512,), 77, dtype=torch.uint8, device="cuda")
    _lib.call("srt_gated_ffn_fwd", C.byref(d), s["x"].data_ptr(), s["wgu"].data_ptr(), s["wd"].data_ptr(), None, y.data_ptr(), scratch.data_ptr(), n, st)
    assert (scratch[n:] == 77).all()
    dx, dw, dd = (torch.full((n + 3, w), 7.0, device="cuda", dtype=BF) for n, w in ((t, c), (2 * f, c), (c, f)))
    n = _lib.lib().srt_gated_ffn_bwd_scratch_bytes(C.byref(d), _lib.SRT_BF16)
    scratch = torch.full((n + 512,), 77, dtype=torch.uint8, device="cuda")
    _lib.call("srt_gated_ffn_bwd", C.byref(d), s["dy"].data_ptr(), s["x"].data_ptr(), s["wgu"].data_ptr(), s["wd"].data_ptr(), _lib.SRT_BF16, dx.data_ptr(),
              dw.data_ptr(), dd.data_ptr(), scratch.data_ptr(), n, st)
    for whole, rows, want in ((y, t, ops.gated_ffn(s["x"], s["wgu"], s["wd"])), (dx, t, None), (dw, 2 * f, None), (dd, c, None)):
        assert (whole[rows:] == 7.0).all() and not (whole[:rows] == 7.0).all()
        if want is not None:
            assert torch.equal(whole[:rows], want)
    assert (scratch[n:] == 77).all()


def test_outputs_that_are_not_wanted():
    t, c, f = 140, 136, 264
    s = make(t, c, f)
    want = ops.gated_ffn_backward(s["dy"], s["x"], s["wgu"], s["wd"])
    d = _lib.GatedFfnDesc(t, c, f)
    n = _lib.lib().srt_gated_ffn_bwd_scratch_bytes(C.byref(d), _lib.SRT_BF16)
    scratch = torch.empty(n, dtype=torch.uint8, device="cuda")
    for k in range(3):
        out = [torch.empty_like(w) if i == k else None for i, w in enumerate(want)]
        _lib.call("srt_gated_ffn_bwd", C.byref(d), s["dy"].data_ptr(), s["x"].data_ptr(), s["wgu"].data_ptr(), s["wd"].data_ptr(), _lib.SRT_BF16,
                  *[None if o is None else o.data_ptr() for o in out], scratch.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
        assert torch.equal(out[k], want[k])


def test_captured_and_replayed_on_two_streams():
    """Forward and backward in two graphs that are replayed side by side, with new inputs copied in; then eagerly again."""
    sizes = [(1, 896, 1064), (300, 136, 1032)]
    sets = [make(*z) for z in sizes]
    want = [(ops.gated_ffn(s["x"], s["wgu"], s["wd"], s["res"]), *ops.gated_ffn_backward(s["dy"], s["x"], s["wgu"], s["wd"])) for s in sets]
    static = [{k: torch.zeros_like(v) for k, v in s.items()} for s in sets]
    graphs, outs = [], []
    for s in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((ops.gated_ffn(s["x"], s["wgu"], s["wd"], s["res"]), *ops.gated_ffn_backward(s["dy"], s["x"], s["wgu"], s["wd"])))
        graphs.append(g)
    for s, z in zip(static, sets):
        for k in s:
            s[k].copy_(z[k])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert ops.tc_status() == 0
    for o, w, s in zip(outs, want, sets):
        assert all(torch.equal(a, b) for a, b in zip(o, w))
        assert torch.equal(ops.gated_ffn(s["x"], s["wgu"], s["wd"], s["res"]), w[0])


def test_two_threads_at_once():
    """Two host threads, each on its own stream, take the same calls as one."""
    import threading
    sets = [make(5, 136, 264), make(600, 136, 1032)]

    def calls(s):
        y, h, rstd = ops.rmsnorm(s["x"], s["gamma"], 1e-6, s["res"])
        return (y, h, rstd, ops.gated_ffn(y, s["wgu"], s["wd"], h), *ops.gated_ffn_backward(s["dy"], y, s["wgu"], s["wd"]),
                ops.grad_norm([s["wgu"], s["wd"]], 1.0))
    for s in sets:
        s["gamma"] = torch.linspace(0.5, 1.5, s["x"].shape[1], device="cuda")
    want = [calls(s) for s in sets]
    torch.cuda.synchronize()
    wrong = []

    def run(s, w):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(100):
                    got = calls(s)
                torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, w)):
                wrong.append("results")
        except Exception as e:
            wrong.append(e)
    threads = [threading.Thread(target=run, args=a) for a in zip(sets, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and ops.tc_status() == 0


# cuts of the plain products: a tile a cluster, of every cluster size there is; token counts at the bounds of the dot products
FEW = [(1, 4096, 11008), (2, 2048, 8192), (2, 2048, 8200), (3, 896, 4864), (4, 896, 4864), (4, 712, 4104), (5, 896, 4864), (16, 2048, 8192),
       (24, 4096, 11008), (33, 5120, 6920), (64, 1536, 8960), (100, 1024, 4096), (128, 896, 1288), (200, 896, 4864), (200, 1544, 8936), (512, 896, 4864),
       (640, 1024, 1096)]


@pytest.mark.parametrize("t,c,f", FEW)
def test_few_tokens_against_long_reductions(t, c, f):
    s = make(t, c, f)
    y = ops.gated_ffn(s["x"], s["wgu"], s["wd"], residual=s["res"])
    got = ops.gated_ffn_backward(s["dy"], s["x"], s["wgu"], s["wd"])
    assert ops.tc_status() == 0
    close(y, *reference(s["x"], s["wgu"], s["wd"], s["res"]), "y")
    want, tol = reference(s["x"], s["wgu"], s["wd"], dy=s["dy"])
    for a, b, e, what in zip(got, want, tol, ("dx", "dw_gate_up", "dw_down")):
        close(a, b, (e + H * (b.abs() + e)) * 1.01, what)
    assert torch.equal(y, ops.gated_ffn(s["x"], s["wgu"], s["wd"], residual=s["res"]))
    assert torch.equal(got[0], ops.gated_ffn_backward(s["dy"], s["x"], s["wgu"], s["wd"])[0])


@pytest.mark.parametrize("t,c,f", [(7, 136, 4104), (24, 896, 4864), (300, 264, 4104)])
def test_bad_tokens_in_shared_tiles(t, c, f):
    """A token that is not a number leaves the other rows of its tile alone."""
    s = make(t, c, f)
    want, dwant = ops.gated_ffn(s["x"], s["wgu"], s["wd"], s["res"]), ops.gated_ffn_backward(s["dy"], s["x"], s["wgu"], s["wd"])[0]
    x = s["x"].clone()
    x[t - 2, 5] = float("nan")
    y, dx = ops.gated_ffn(x, s["wgu"], s["wd"], s["res"]), ops.gated_ffn_backward(s["dy"], x, s["wgu"], s["wd"])[0]
    good = torch.arange(t, device="cuda") != t - 2
    assert torch.equal(y[good], want[good]) and torch.equal(dx[good], dwant[good]) and y[t - 2].isnan().all()
