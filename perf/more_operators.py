"""The timed work of the dense side of a layer and of the step that trains it, as a program
calls them:

- "product": a matrix product with its bias, activation and residual in the epilogue
  (`dense.product`), and its backward (`dense.product_backward`: the gradients to the rows, the
  kernel and the bias);
- "block": a dense feed-forward block, gated (up and gate projections, the activation and their
  product) or plain, its down product and the residual's addition (`mlp.feed_forward`), and a
  training step of it (`mlp.feed_forward_backward` after it);
- "clip": the global norm of a layer's gradients and their clipping by it (`clip.clipped`).

Where `own` is false, `run` computes them in plain form, by elementary torch operations in
float32 (float64 in the norm's long sum), rounded once at the end.
"""

import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def _product(**kw):
    return {"kind": "product", "direction": "forward", "dtype": "bfloat16", "activation": "none",
            "bias": False, "residual": False, **kw}


def _block(**kw):
    return {"kind": "block", "direction": "forward", "dtype": "bfloat16", "activation": "swish",
            "gated": True, "bias": False, "residual": False, "limit": 0.0, "offset": 0.0, **kw}


def _clip(**kw):
    return {"kind": "clip", "dtype": "bfloat16", "clips": True, **kw}


def listed():
    return [
        # a decode step of one sequence: attention's output projection onto the residual stream
        _product(name="product one token", m=1, k=4096, n=4096, residual=True),
        # a decode batch's, with a bias, into a width of gpt-oss-120b's
        _product(name="product decode 48", m=48, k=4096, n=2880, bias=True, residual=True),
        # a long prompt through a plain up projection (DeepSeek-V3's width)
        _product(name="product prompt", m=8192, k=7168, n=4096, bias=True,
                 activation="gelu_tanh"),
        # a small float32 layer, odd in every dimension
        _product(name="product odd float32", m=1001, k=1443, n=1027, dtype="float32", bias=True,
                 activation="swish", residual=True),
        # the backward of a projection with its bias and activation over a training batch
        _product(name="product backward", m=16384, k=2048, n=4096, direction="backward",
                 bias=True, activation="gelu_tanh"),
        # the shared expert (DeepSeek-V3's width and units) for one token
        _block(name="block one token", m=1, d=7168, f=2048, residual=True),
        # a decode batch or a short prompt through a clamped block with biases
        _block(name="block decode 201", m=201, d=2880, f=2880, bias=True, residual=True,
               limit=7.0, offset=1.0),
        # a long prompt through the shared expert
        _block(name="block prompt", m=8192, d=7168, f=2048, residual=True),
        # a training step of a dense block over a whole batch, forward and backward
        _block(name="block step", m=16384, d=2048, f=8192, direction="step"),
        # a small step, odd in every dimension, with biases
        _block(name="block step odd", m=1501, d=1027, f=771, direction="step", bias=True),
        # a small model's gradients in float32: a launch's latency
        _clip(name="clip small", d=256, f=512, experts=8, dtype="float32"),
        # a layer of Qwen3-30B-A3B's gradients: its experts', its router's and its norm's
        _clip(name="clip layer", d=2048, f=768, experts=128),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi, odd):
    n = _log_int(rng, lo, hi)
    return n if odd else max(lo, n // 16 * 16)


def draw(rng):
    kind = rng.choice(["product", "product", "block", "block", "clip"])
    if kind == "clip":
        d, f = _log_int(rng, 64, 4096), _log_int(rng, 64, 4096)
        experts = _log_int(rng, 1, max(1, min(128, 600_000_000 // (3 * d * f))))
        return _clip(d=d, f=f, experts=experts, dtype=rng.choice(["bfloat16", "float32"])
                     if experts * d * f < 60_000_000 else "bfloat16", clips=rng.random() < 0.8)
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    most = 3.0e11 if dtype == "float32" else 2.0e12
    odd = rng.random() < 0.3
    if kind == "product":
        backward = rng.random() < 0.4
        k, n = _width(rng, 64, 8192, odd), _width(rng, 64, 8192, odd)
        rows = int(most / ((6 if backward else 2) * k * n))
        return _product(m=_log_int(rng, 1, max(1, min(16384, rows))), k=k, n=n, dtype=dtype,
                        direction="backward" if backward else "forward",
                        bias=rng.random() < 0.5, residual=not backward and rng.random() < 0.5,
                        activation=rng.choice(["none", "swish", "gelu", "gelu_tanh", "relu2"]))
    step = rng.random() < 0.5
    d, f = _width(rng, 64, 8192, odd), _width(rng, 64, 8192, odd)
    gated = rng.random() < 0.8
    rows = int(most / ((6 if gated else 4) * (3 if step else 1) * d * f))
    limit = rng.choice([0.0, 0.0, 7.0])
    return _block(m=_log_int(rng, 1, max(1, min(16384, rows))), d=d, f=f, dtype=dtype, gated=gated,
                  direction="step" if step else "forward", bias=rng.random() < 0.4,
                  activation=rng.choice(["swish", "swish", "gelu", "gelu_tanh"]),
                  residual=rng.random() < 0.5, limit=limit,
                  offset=1.0 if gated and limit else 0.0)


# --- inputs ------------------------------------------------------------------------------


def _dtype(case):
    return F32 if case["dtype"] == "float32" else BF16


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _kernel(gen, dt, rows, *cols):
    """A kernel as a trained layer has it: its products of N(0, 1) rows are of order 1."""
    return (_randn(gen, rows, *cols) / math.sqrt(rows)).to(dt)


def _inputs(case, seed):
    """The case's inputs, by name."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _dtype(case)
    if case["kind"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        x = {"x": _randn(gen, m, k).to(dt), "w": _kernel(gen, dt, k, n),
             "b": (0.5 * _randn(gen, n)).to(dt) if case["bias"] else None}
        if case["direction"] == "forward":
            x["residual"] = _randn(gen, m, n).to(dt) if case["residual"] else None
            return x
        x["dy"] = (0.01 * _randn(gen, m, n)).to(dt)
        # what the forward kept: the product before its activation
        kept = x["x"].float() @ x["w"].float()
        x["product"] = None if case["activation"] == "none" else (
            kept if x["b"] is None else kept + x["b"].float()).to(dt)
        return x
    if case["kind"] == "block":
        m, d, f, p = case["m"], case["d"], case["f"], 2 if case["gated"] else 1
        return {"x": _randn(gen, m, d).to(dt), "up": _kernel(gen, dt, d, f, p),
                "down": _kernel(gen, dt, f, d),
                "up_bias": (0.5 * _randn(gen, f, p)).to(dt) if case["bias"] else None,
                "down_bias": (0.5 * _randn(gen, d)).to(dt) if case["bias"] else None,
                "residual": _randn(gen, m, d).to(dt) if case["residual"] else None,
                "dy": (0.01 * _randn(gen, m, d)).to(dt) if case["direction"] == "step" else None}
    # a layer's gradients: its experts' up and down, its router's kernel, and in float32 the
    # router's bias and two norms' gains (they are sums)
    d, f, e = case["d"], case["f"], case["experts"]
    grads = [torch.empty(s, dtype=dt, device="cuda")
             for s in ((e, d, f, 2), (e, f, d), (d, e))]
    for g in grads:  # a slice at a time: they are large
        for part in g:
            part.copy_(1e-3 * _randn(gen, *part.shape))
    grads += [1e-2 * _randn(gen, n) for n in (e, d, d)]
    count = sum(g.numel() for g in grads)
    # the norm is about 1e-3 sqrt(count): a limit of a tenth of it clips, of ten times does not
    return {"grads": grads, "max_norm": 1e-3 * math.sqrt(count) * (0.1 if case["clips"] else 10.0)}


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


# --- the operators in plain form -----------------------------------------------------------


def _activated(kind, z):
    if kind == "swish":
        return z * torch.sigmoid(z)
    if kind == "gelu":
        return z * 0.5 * torch.erfc(z * -math.sqrt(0.5))
    if kind == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
    if kind == "relu2":
        return torch.relu(z).square()
    return z


def _slope(kind, z):
    """The activation's derivative."""
    if kind == "swish":
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    if kind == "gelu":
        return 0.5 * torch.erfc(z * -math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) / math.sqrt(
            2 * math.pi)
    if kind == "gelu_tanh":
        c = 2 * math.sqrt(2 / math.pi)
        s = torch.sigmoid(c * (z + 0.044715 * z * z * z))
        return s + z * s * (1 - s) * c * (1 + 3 * 0.044715 * z * z)
    if kind == "relu2":
        return 2 * torch.relu(z)
    return torch.ones_like(z)


def _plain_product(s):
    case, dt = s["case"], s["x"].dtype
    if case["direction"] == "backward":
        dz = s["dy"].float()
        if s["product"] is not None:
            dz = dz * _slope(case["activation"], s["product"].float())
        return {"x": (dz @ s["w"].float().T).to(dt), "w": (s["x"].float().T @ dz).to(dt),
                "bias": dz.sum(0).to(dt) if s["b"] is not None else None}
    y = s["x"].float() @ s["w"].float()
    if s["b"] is not None:
        y = y + s["b"].float()
    y = _activated(case["activation"], y)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"out": y.to(dt)}


def _plain_block(s):
    case, dt = s["case"], s["x"].dtype
    m, d, f, p = case["m"], case["d"], case["f"], 2 if case["gated"] else 1
    kind, limit = case["activation"], case["limit"]
    x, up, down = s["x"].float(), s["up"].float().view(d, f * p), s["down"].float()
    z = x @ up
    if s["up_bias"] is not None:
        z = z + s["up_bias"].float().view(-1)
    z = z.view(m, f, p)
    u, g = z[..., 0], z[..., -1]
    cu = u.clamp(-limit, limit) if limit else u
    if case["gated"]:
        cg = g.clamp(max=limit) if limit else g
        h = _activated(kind, cg) * (cu + case["offset"])
    else:
        h = _activated(kind, cu)
    y = h @ down
    if s["down_bias"] is not None:
        y = y + s["down_bias"].float()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"out": y.to(dt)}
    if case["direction"] == "forward":
        return out
    dy = s["dy"].float()
    dh = dy @ down.T
    inside = (u.abs() < limit).float() if limit else 1.0
    if case["gated"]:
        below = (g < limit).float() if limit else 1.0
        dp = torch.stack([dh * _activated(kind, cg) * inside,
                          dh * (cu + case["offset"]) * _slope(kind, cg) * below], -1)
    else:
        dp = (dh * _slope(kind, cu) * inside)[..., None]
    dp = dp.view(m, f * p)
    out.update(x=(dp @ up.T).to(dt), up=(x.T @ dp).view(d, f, p).to(dt), down=(h.T @ dy).to(dt))
    if s["up_bias"] is not None:
        out.update(up_bias=dp.sum(0).view(f, p).to(dt), down_bias=dy.sum(0).to(dt))
    return out


def _plain_clip(s):
    total = sum(g.double().square().sum() for g in s["grads"])
    norm = total.sqrt()
    factor = (s["max_norm"] / norm).clamp(max=1.0).float()
    return {"norm": norm.float(), "grads": [(g.float() * factor).to(g.dtype) for g in s["grads"]]}


def _plain(s):
    kind = s["case"]["kind"]
    return (_plain_product if kind == "product" else _plain_block if kind == "block"
            else _plain_clip)(s)


# --- the framework's -------------------------------------------------------------------------


def _call(s):
    case = s["case"]
    if case["kind"] == "product":
        from bux_amd import dense
        activation = None if case["activation"] == "none" else case["activation"]
        if case["direction"] == "backward":
            g = dense.product_backward(s["dy"], s["x"], s["w"], activation=activation,
                                       product=s["product"], bias=case["bias"])
            return {"x": g.x, "w": g.w, "bias": g.bias}
        return {"out": dense.product(s["x"], s["w"], bias=s["b"], activation=activation,
                                     residual=s["residual"]).out}
    if case["kind"] == "block":
        from bux_amd import mlp, moe
        ffn = moe.Ffn(case["activation"], case["limit"] or None, case["offset"])
        step = case["direction"] == "step"
        r = mlp.feed_forward(s["x"], s["up"], s["down"], ffn, up_bias=s["up_bias"],
                             down_bias=s["down_bias"], residual=s["residual"], keep=step)
        if not step:
            return {"out": r.out}
        g = mlp.feed_forward_backward(s["dy"], r.saved, s["up"], s["down"], ffn,
                                      bias=case["bias"])
        out = {"out": r.out, "x": g.x, "up": g.up, "down": g.down}
        if case["bias"]:
            out.update(up_bias=g.up_bias, down_bias=g.down_bias)
        return out
    from bux_amd import clip
    r = clip.clipped(s["grads"], s["max_norm"])
    return {"norm": r.norm, "grads": r.grads}


def run(state):
    if own:
        return _call(state)
    return _plain(state)


# --- what a pass cannot do without --------------------------------------------------------


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        if case["direction"] == "forward":
            return {"bytes": size * (m * k + k * n + m * n * (2 if case["residual"] else 1)
                                     + (n if case["bias"] else 0)), "flops": 2 * m * k * n}
        kept = 0 if case["activation"] == "none" else m * n
        return {"bytes": size * (2 * m * k + 2 * k * n + m * n + kept
                                 + (n if case["bias"] else 0)), "flops": 4 * m * k * n}
    if case["kind"] == "block":
        m, d, f, p = case["m"], case["d"], case["f"], 2 if case["gated"] else 1
        weights = (p + 1) * d * f
        biases = p * f + d if case["bias"] else 0
        tokens = m * d * (3 if case["residual"] else 2)
        if case["direction"] == "forward":
            return {"bytes": size * (weights + tokens + biases), "flops": 2 * m * weights}
        return {"bytes": size * (2 * weights + tokens + 2 * m * d + 2 * biases), "flops": 6 * m * weights}
    d, f, e = case["d"], case["f"], case["experts"]
    values, sums = 3 * e * d * f + d * e, e + 2 * d
    return {"bytes": 2 * (size * values + 4 * sums) + 4, "flops": 3 * (values + sums)}


# --- in 64 bits ------------------------------------------------------------------------------


def _phi(kind, z):
    """The activation and its derivative, by their definitions."""
    if kind == "swish":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if kind == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        dt = (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 0.134145 * z * z)
        return z * (1 + t) / 2, (1 + t) / 2 + z * dt / 2
    if kind == "relu2":
        r = torch.where(z > 0, z, 0.0)
        return r * r, 2 * r
    return z, torch.ones_like(z)


def _mm(a, b):
    return torch.mm(a.contiguous(), b.contiguous())


def _exact_product(case, x):
    a, w = x["x"].to(F64), x["w"].to(F64)
    if case["direction"] == "backward":
        dz = x["dy"].to(F64)
        if x["product"] is not None:
            dz = dz * _phi(case["activation"], x["product"].to(F64))[1]
        return {"x": _mm(dz, w.t()), "w": _mm(a.t(), dz),
                "bias": None if x["b"] is None else dz.sum(0)}
    z = _mm(a, w)
    if x["b"] is not None:
        z += x["b"].to(F64)
    y = _phi(case["activation"], z)[0]
    return {"out": y if x["residual"] is None else y + x["residual"].to(F64)}


def _exact_block(case, x):
    d, f = case["d"], case["f"]
    limit = case["limit"] or math.inf
    a, up, down = x["x"].to(F64), x["up"].to(F64), x["down"].to(F64)
    # the up and the gate projection, each as a product of its own
    parts = [_mm(a, up[..., i]) for i in range(up.shape[2])]
    if x["up_bias"] is not None:
        parts = [z + x["up_bias"].to(F64)[:, i] for i, z in enumerate(parts)]
    u = torch.maximum(torch.minimum(parts[0], torch.full_like(parts[0], limit)),
                      torch.full_like(parts[0], -limit))
    if case["gated"]:
        g = torch.minimum(parts[1], torch.full_like(u, limit))
        act, slope = _phi(case["activation"], g)
        h = act * (u + case["offset"])
    else:
        h, slope = _phi(case["activation"], u)
    y = _mm(h, down)
    for extra in (x["down_bias"], x["residual"]):
        if extra is not None:
            y += extra.to(F64)
    out = {"out": y}
    if case["direction"] == "forward":
        return out
    dy = x["dy"].to(F64)
    dh = _mm(dy, down.t())
    free = (parts[0].abs() < limit).to(F64)
    if case["gated"]:
        dps = [dh * act * free, dh * (u + case["offset"]) * slope * (parts[1] < limit)]
    else:
        dps = [dh * slope * free]
    out["x"] = sum(_mm(dp, up[..., i].t()) for i, dp in enumerate(dps))
    out["up"] = torch.stack([_mm(a.t(), dp) for dp in dps], -1)
    out["down"] = _mm(h.t(), dy)
    if x["up_bias"] is not None:
        out["up_bias"] = torch.stack([dp.sum(0) for dp in dps], -1)
        out["down_bias"] = dy.sum(0)
    return out


def _exact_clip(case, x):
    squares = [torch.stack([part.to(F64).pow(2).sum() for part in g.split(max(1, g.shape[0] // 8))])
               .sum() for g in x["grads"]]
    norm = torch.stack(squares).sum().sqrt()
    factor = torch.where(norm > x["max_norm"], x["max_norm"] / norm, 1.0)
    return {"norm": norm, "grads": [g.to(F64) * factor for g in x["grads"]]}


def exact(case, seed):
    x = _inputs(case, seed)
    return (_exact_product if case["kind"] == "product" else _exact_block
            if case["kind"] == "block" else _exact_clip)(case, x)
