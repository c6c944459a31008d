"""The work that the operators of a decoder's feed-forward half and of its optimizer step are judged by.

Three operators, each with its directions and types: the gated feed-forward block (`ops.gated_ffn`,
`ops.gated_ffn_backward`, `ops.gated_ffn_e4m3`), the root-mean-square norm with the residual's addition (`ops.rmsnorm`,
`ops.rmsnorm_e4m3`, `ops.rmsnorm_backward`), and the global gradient norm with clipping (`ops.clip_grad_norm`, and
`ops.grad_norm` with the AdamW step that takes the coefficient). With `own` false the same values are computed from
elementary torch operations in 32 bits.
"""
import math

import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0
ADAMW = dict(lr=3e-4, b1=0.9, b2=0.999, eps=1e-8, wd=0.01, step=10)
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one generated token through the feed-forward half of the grouped-query decoder: weights are streamed once
        {"name": "ffn_token", "kind": "ffn_fwd", "tokens": 1, "width": 896, "hidden": 4864},
        # the decoder's training micro-batch, 4 sequences of 2048
        {"name": "ffn_train_4x2048", "kind": "ffn_fwd", "tokens": 8192, "width": 896, "hidden": 4864},
        # ragged sequences packed together, through a wider block whose widths are no multiples of a tile
        {"name": "ffn_ragged_1237", "kind": "ffn_fwd", "tokens": 1237, "width": 1544, "hidden": 8936},
        # backward of the training micro-batch, and of one short sequence
        {"name": "ffn_backward_4x2048", "kind": "ffn_bwd", "tokens": 8192, "width": 896, "hidden": 4864},
        {"name": "ffn_backward_333", "kind": "ffn_bwd", "tokens": 333, "width": 896, "hidden": 4864},
        # 24 requests answered together from weights in 8 bits, one token each
        {"name": "ffn_e4m3_24", "kind": "ffn_e4m3", "tokens": 24, "width": 4096, "hidden": 11008},
        # the norm between the halves of a decoder layer, training
        {"name": "norm_train_4x2048", "kind": "norm_fwd", "tokens": 8192, "width": 896, "type": "bf16"},
        # the same in full precision at an odd size
        {"name": "norm_f32_777", "kind": "norm_fwd", "tokens": 777, "width": 2056, "type": "f32"},
        # what feeds the 8-bit block above
        {"name": "norm_e4m3_24", "kind": "norm_e4m3", "tokens": 24, "width": 4096, "type": "bf16"},
        {"name": "norm_backward_4x2048", "kind": "norm_bwd", "tokens": 8192, "width": 896, "type": "bf16"},
        # every gradient of the grouped-query decoder, clipped in place (169 tensors, 0.49 G elements)
        {"name": "clip_169_tensors", "kind": "clip", "layers": 24, "width": 896, "hidden": 4864, "vocab": 151936, "type": "f32", "padded": True},
        # norm, clipping and AdamW on the flat buffers of the small decoder (124 M parameters)
        {"name": "clip_adamw_124m", "kind": "clip_adamw", "count": 124439808},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["ffn_fwd", "ffn_fwd", "ffn_bwd", "ffn_e4m3", "norm_fwd", "norm_e4m3", "norm_bwd", "clip", "clip_adamw"])
    if kind.startswith("ffn"):
        unit = 16 if kind == "ffn_e4m3" else 8
        width, hidden = unit * _log_int(rng, 256 // unit, 4096 // unit), 8 * _log_int(rng, 64, 1376)
        most = (8192 * 896 * 4864) // (width * hidden)
        return {"kind": kind, "tokens": _log_int(rng, 1, max(1, min(8192, most))), "width": width, "hidden": hidden}
    if kind.startswith("norm"):
        width = 8 * _log_int(rng, 8, 1024)
        return {"kind": kind, "tokens": _log_int(rng, 1, max(1, min(16384, 8192 * 896 // width))), "width": width, "type": rng.choice(["bf16", "f32"])}
    if kind == "clip":
        return {"kind": kind, "layers": rng.randint(1, 40), "width": _log_int(rng, 33, 1024), "hidden": _log_int(rng, 65, 2048), "vocab": _log_int(rng, 100, 50257),
                "type": rng.choice(["bf16", "f32"]), "padded": rng.random() < 0.5}
    return {"kind": kind, "count": _log_int(rng, 10000, 124439808)}


def _tensor_sizes(case):
    """The gradients of a decoder: the token table, then per layer two norms, the attention's projections and the block's three matrices."""
    w, f = case["width"], case["hidden"]
    return [case["vocab"] * w] + [w, 2 * w * w, w * w, w, w * f, w * f, f * w] * case["layers"]


def _starts(case):
    """Where each tensor begins in the flat buffer: on multiples of 64 elements where the buffer is padded, else back to back. The last entry is the length."""
    at = [0]
    for n in _tensor_sizes(case):
        at.append(at[-1] + (-(-n // 64) * 64 if case["padded"] else n))
    return at


def _quantise(x):
    """Rows to 8 bits as a program does that loads a checkpoint: the largest value of a row becomes 448."""
    scale = x.float().abs().amax(-1) / E4M3_MAX
    return (x.float() / scale[:, None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(0.0, std, generator=gen).to(dtype)

    if kind.startswith("ffn"):
        t, c, f = case["tokens"], case["width"], case["hidden"]
        s = {"kind": kind, "x": normal(t, c), "w_gate_up": normal(2 * f, c, std=0.02), "w_down": normal(c, f, std=0.02)}
        if kind == "ffn_bwd":
            s["dy"] = normal(t, c, std=1e-3)
        else:
            s["residual"] = normal(t, c)
        if kind == "ffn_e4m3":
            s["x"], s["x_scale"] = _quantise(s["x"])
            s["w_gate_up"], s["w_scale"] = _quantise(s["w_gate_up"])
        return s
    if kind.startswith("norm"):
        t, c, dtype = case["tokens"], case["width"], TYPES[case["type"]]
        s = {"kind": kind, "x": normal(t, c, std=2.0, dtype=dtype), "gamma": 1.0 + normal(c, std=0.1, dtype=torch.float32)}
        if kind == "norm_bwd":
            s["dy"], s["dh"] = normal(t, c, std=1e-3, dtype=dtype), normal(t, c, std=1e-3, dtype=dtype)
            s["rstd"] = (1.0 / (s["x"].double().square().mean(-1) + EPS).sqrt()).float()
        else:
            s["residual"] = normal(t, c, std=2.0, dtype=dtype)
        return s
    if kind == "clip":
        at, sizes = _starts(case), _tensor_sizes(case)
        flat = torch.zeros(at[-1], device="cuda", dtype=TYPES[case["type"]])
        grads = [flat[a:a + n] for a, n in zip(at, sizes)]
        for g in grads:
            g.copy_(torch.empty(g.numel(), device="cuda").normal_(0.0, 1e-3, generator=gen))
        # what a step that has to be clipped meets: a norm of several times the bound
        return {"kind": kind, "flat": flat, "grads": grads, "max_norm": 1e-3 * math.sqrt(sum(sizes)) / 4.0}
    n = case["count"]
    f32 = dict(dtype=torch.float32)
    return {"kind": kind, "p": normal(n, std=0.02, **f32), "g": normal(n, std=1e-3, **f32), "m": normal(n, std=1e-4, **f32),
            "v": normal(n, std=1e-4, **f32).square_(), "p_bf16": torch.empty(n, device="cuda", dtype=torch.bfloat16), "max_norm": 1.0}


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from sirius_b200 import ops
    kind = s["kind"]
    if kind == "ffn_fwd":
        return {"y": ops.gated_ffn(s["x"], s["w_gate_up"], s["w_down"], residual=s["residual"])}
    if kind == "ffn_e4m3":
        return {"y": ops.gated_ffn_e4m3(s["x"], s["x_scale"], s["w_gate_up"], s["w_scale"], s["w_down"], residual=s["residual"])}
    if kind == "ffn_bwd":
        dx, dw_gate_up, dw_down = ops.gated_ffn_backward(s["dy"], s["x"], s["w_gate_up"], s["w_down"])
        return {"dx": dx, "dw_gate_up": dw_gate_up, "dw_down": dw_down}
    if kind == "norm_fwd":
        y, h, rstd = ops.rmsnorm(s["x"], s["gamma"], EPS, residual=s["residual"])
        return {"y": y, "h": h, "rstd": rstd}
    if kind == "norm_e4m3":
        q, scale, h, rstd = ops.rmsnorm_e4m3(s["x"], s["gamma"], EPS, residual=s["residual"])
        return {"q": q, "scale": scale, "h": h, "rstd": rstd}
    if kind == "norm_bwd":
        dx, dgamma = ops.rmsnorm_backward(s["dy"], s["x"], s["gamma"], s["rstd"], dh=s["dh"])
        return {"dx": dx, "dgamma": dgamma}
    if kind == "clip":
        return {"norm": ops.clip_grad_norm(s["grads"], s["max_norm"])[0], "grads": s["flat"]}
    clip = ops.grad_norm([s["g"]], s["max_norm"])
    ops.adamw(s["p"], s["g"], s["m"], s["v"], ADAMW["lr"], ADAMW["b1"], ADAMW["b2"], ADAMW["eps"], ADAMW["wd"], ADAMW["step"], p_bf16=s["p_bf16"], clip=clip)
    return {"norm": clip[0], "p": s["p"], "m": s["m"], "v": s["v"], "p_bf16": s["p_bf16"]}


def _plain(s):
    kind = s["kind"]
    if kind.startswith("ffn"):
        x, wgu, wd = s["x"].float(), s["w_gate_up"].float(), s["w_down"].float()
        if kind == "ffn_e4m3":
            x, wgu = x * s["x_scale"][:, None], wgu * s["w_scale"][:, None]
        f = wd.shape[1]
        gu = x @ wgu.T
        gate, up = gu[:, :f], gu[:, f:]
        sig = 1.0 / (1.0 + torch.exp(-gate))
        silu = gate * sig
        act = silu * up
        if kind != "ffn_bwd":
            return {"y": (s["residual"].float() + act @ wd.T).to(s["residual"].dtype)}
        dy = s["dy"].float()
        dact = dy @ wd
        dgu = torch.cat([dact * up * (sig + silu * (1.0 - sig)), dact * silu], dim=1)
        return {"dx": (dgu @ wgu).to(s["x"].dtype), "dw_gate_up": (dgu.T @ x).to(s["x"].dtype), "dw_down": (dy.T @ act).to(s["x"].dtype)}
    if kind.startswith("norm"):
        x, gamma = s["x"].float(), s["gamma"]
        if kind == "norm_bwd":
            xhat, g = x * s["rstd"][:, None], s["dy"].float() * gamma
            dx = s["dh"].float() + s["rstd"][:, None] * (g - xhat * (g * xhat).mean(-1, keepdim=True))
            return {"dx": dx.to(s["x"].dtype), "dgamma": (s["dy"].float() * xhat).sum(0)}
        h = x + s["residual"].float()
        rstd = 1.0 / torch.sqrt((h * h).mean(-1) + EPS)
        y = h * rstd[:, None] * gamma
        h = h.to(s["x"].dtype)
        if kind == "norm_fwd":
            return {"y": y.to(s["x"].dtype), "h": h, "rstd": rstd}
        # values next to a rounding border: in 64 bits up to the rounding
        wide = s["x"].double() + s["residual"].double()
        wide = wide / torch.sqrt((wide * wide).mean(-1, keepdim=True) + EPS) * gamma.double()
        scale = wide.abs().amax(-1) / E4M3_MAX
        return {"q": (wide / scale[:, None]).float().to(torch.float8_e4m3fn), "scale": scale.float(), "h": h, "rstd": rstd}
    if kind == "clip":
        norm = (s["flat"].double() * s["flat"].double()).sum().sqrt()
        coefficient = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
        s["flat"].copy_(s["flat"].float() * coefficient.float())
        return {"norm": norm.float(), "grads": s["flat"]}
    norm = (s["g"].double() * s["g"].double()).sum().sqrt()
    g = s["g"] * torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0).float()
    a = ADAMW
    s["p"].copy_(s["p"] * (1.0 - a["lr"] * a["wd"]))
    s["m"].copy_(a["b1"] * s["m"] + (1.0 - a["b1"]) * g)
    s["v"].copy_(a["b2"] * s["v"] + (1.0 - a["b2"]) * g * g)
    denominator = torch.sqrt(s["v"]) / math.sqrt(1.0 - a["b2"] ** a["step"]) + a["eps"]
    s["p"].copy_(s["p"] - a["lr"] / (1.0 - a["b1"] ** a["step"]) * (s["m"] / denominator))
    s["p_bf16"].copy_(s["p"])
    return {"norm": norm.float(), "p": s["p"], "m": s["m"], "v": s["v"], "p_bf16": s["p_bf16"]}


def exact(case, seed):
    """The definitions in 64 bits: y = residual + W_down (silu(W_gate x) * W_up x) and its derivatives, y_i = gamma_i h_i / rms(h), and gradients
    scaled by min(1, bound / norm). The 8-bit output has no value here: it is a choice between neighbours, not a number."""
    s = prepare(case, seed)
    kind = case["kind"]
    if kind.startswith("ffn"):
        f = case["hidden"]
        x = s["x"].to(torch.float64)
        gate_w, up_w = s["w_gate_up"][:f].to(torch.float64), s["w_gate_up"][f:].to(torch.float64)
        down = s["w_down"].to(torch.float64)
        if kind == "ffn_e4m3":
            x = torch.einsum("tc,t->tc", x, s["x_scale"].to(torch.float64))
            gate_w = torch.einsum("fc,f->fc", gate_w, s["w_scale"][:f].to(torch.float64))
            up_w = torch.einsum("fc,f->fc", up_w, s["w_scale"][f:].to(torch.float64))
        a, b = torch.einsum("tc,fc->tf", x, gate_w), torch.einsum("tc,fc->tf", x, up_w)
        s1 = torch.sigmoid(a)
        if kind != "ffn_bwd":
            return {"y": s["residual"].to(torch.float64) + torch.einsum("tf,cf->tc", a * s1 * b, down)}
        dy = s["dy"].to(torch.float64)
        d = torch.einsum("tc,cf->tf", dy, down)
        da, db = d * b * s1 * (1.0 + a * (1.0 - s1)), d * a * s1
        return {"dx": torch.einsum("tf,fc->tc", da, gate_w) + torch.einsum("tf,fc->tc", db, up_w),
                "dw_gate_up": torch.cat([torch.einsum("tf,tc->fc", da, x), torch.einsum("tf,tc->fc", db, x)]),
                "dw_down": torch.einsum("tc,tf->cf", dy, a * s1 * b)}
    if kind.startswith("norm"):
        gamma, x = s["gamma"].to(torch.float64), s["x"].to(torch.float64)
        if kind == "norm_bwd":
            r, dy = s["rstd"].to(torch.float64).unsqueeze(1), s["dy"].to(torch.float64)
            inner = torch.einsum("tc,tc,c->t", dy, x, gamma).unsqueeze(1) / x.shape[1]
            return {"dx": s["dh"].to(torch.float64) + r * dy * gamma - r ** 3 * inner * x, "dgamma": torch.einsum("tc,tc,t->c", dy, x, r[:, 0])}
        h = torch.add(x, s["residual"].to(torch.float64))
        rstd = torch.rsqrt(torch.linalg.vector_norm(h, dim=1).pow(2) / h.shape[1] + EPS)
        y = torch.einsum("tc,t,c->tc", h, rstd, gamma)
        if kind == "norm_e4m3":
            return {"q": None, "scale": torch.linalg.vector_norm(y, ord=float("inf"), dim=1) / E4M3_MAX, "h": h, "rstd": rstd}
        return {"y": y, "h": h, "rstd": rstd}
    if kind == "clip":
        wide = s["flat"].to(torch.float64)
        norm = torch.linalg.vector_norm(wide)
        return {"norm": norm, "grads": wide * min(1.0, s["max_norm"] / (float(norm) + 1e-6))}
    g = s["g"].to(torch.float64)
    norm = torch.linalg.vector_norm(g)
    g = g * min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    a = ADAMW
    m = torch.lerp(g, s["m"].to(torch.float64), a["b1"])
    v = torch.lerp(g.square(), s["v"].to(torch.float64), a["b2"])
    p = s["p"].to(torch.float64)
    update = (m / (1.0 - a["b1"] ** a["step"])) / ((v / (1.0 - a["b2"] ** a["step"])).sqrt() + a["eps"])
    p = p - a["lr"] * (a["wd"] * p + update)
    return {"norm": norm, "p": p, "m": m, "v": v, "p_bf16": p}


def work(case):
    kind = case["kind"]
    if kind.startswith("ffn"):
        t, c, f = case["tokens"], case["width"], case["hidden"]
        if kind == "ffn_bwd":  # x, dy and dx; weights and their gradients; gate, up and the product's gradient, then dx and three weight gradients
            return {"bytes": 2 * (3 * t * c + 2 * 3 * c * f), "flops": 16 * t * c * f}
        if kind == "ffn_e4m3":
            return {"bytes": t * (c + 4) + 2 * f * (c + 4) + 2 * c * f + 4 * t * c, "flops": 6 * t * c * f}
        return {"bytes": 2 * (3 * t * c + 3 * c * f), "flops": 6 * t * c * f}
    if kind.startswith("norm"):
        t, c = case["tokens"], case["width"]
        e = 4 if case["type"] == "f32" else 2
        if kind == "norm_fwd":    # x and residual; h, y
            return {"bytes": 4 * t * c * e + 4 * c + 4 * t, "flops": 5 * t * c}
        if kind == "norm_e4m3":   # x and residual; h, q and scales
            return {"bytes": 3 * t * c * e + t * c + 4 * c + 8 * t, "flops": 7 * t * c}
        return {"bytes": 4 * t * c * e + 8 * c + 4 * t, "flops": 10 * t * c}
    if kind == "clip":
        n = sum(_tensor_sizes(case))
        return {"bytes": 2 * n * (4 if case["type"] == "f32" else 2), "flops": 3 * n}
    return {"bytes": 30 * case["count"], "flops": 20 * case["count"]}
