"""The dense products' formulas in float64, with the error that their kernels may make.

Each value comes with a bound: the inputs' own errors through the formula, float32 sums of K
products (at most K + 8 roundings of U = 2^-24, relative to the sum of the magnitudes), the
activation's few float32 operations (16 of them, relative to the larger of 1 and what they work
on), and a half step of the output's type (eps / 2 of the value). No bound looks at a result.
"""

import math

import torch

U = 2.0 ** -24
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


class V:
    """float64 values and a bound on how far a kernel's may lie from them."""

    def __init__(self, v, e=None):
        self.v = v.to(F64)
        self.e = torch.zeros_like(self.v) if e is None else e

    def t(self):
        return V(self.v.t(), self.e.t())

    def __matmul__(self, o):
        a, b = self.v.contiguous(), o.v.contiguous()
        k = a.shape[-1]
        mag = a.abs() @ b.abs()
        e = self.e @ (b.abs() + o.e) + a.abs() @ o.e
        return V(a @ b, e + (k + 8) * U * (mag + e))

    def __add__(self, o):
        if o is None:
            return self
        v = self.v + o.v
        e = self.e + o.e
        return V(v, e + 2 * U * (v.abs() + e))

    def sum0(self):
        n = self.v.shape[0]
        return V(self.v.sum(0), self.e.sum(0) + (n + 8) * U * (self.v.abs() + self.e).sum(0))

    def rounded(self, dtype):
        """As one rounding to `dtype` leaves it (the smallest subnormals aside)."""
        half = torch.finfo(dtype).eps / 2
        return V(self.v, self.e + half * (self.v.abs() + self.e) + 1e-37)

    def holds(self, got, what):
        assert tuple(got.shape) == tuple(self.v.shape), (what, got.shape, self.v.shape)
        over = (got.to(F64).to(self.v.device) - self.v).abs() - self.e
        assert torch.isfinite(got).all() or not torch.isfinite(self.v).all(), what
        worst = over.max().item() if over.numel() else -1.0
        assert worst <= 0, (what, worst, over.argmax().item())


def _sigmoid(x):
    return torch.sigmoid(x)


def activation(kind, x, dtype):
    """a(x), its derivative and a bound on the second derivative, in float64."""
    if kind == "swish" or kind == "quick_gelu":
        c = 1.0 if kind == "swish" else (1.703125 if dtype == BF16 else 1.702)
        s = _sigmoid(c * x)
        return x * s, s + c * x * s * (1 - s), torch.full_like(x, 0.55 * c)
    if kind == "relu":
        return torch.relu(x), (x > 0).to(F64), torch.zeros_like(x)
    if kind == "relu2":
        return torch.relu(x) ** 2, 2 * torch.relu(x), torch.full_like(x, 2.0)
    if kind == "gelu":
        cdf = torch.special.ndtr(x)
        pdf = torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
        return x * cdf, cdf + x * pdf, torch.full_like(x, 0.8)
    if kind == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (x + 0.044715 * x ** 3))
        d = (1 + t) / 2 + x / 2 * (1 - t * t) * c * (1 + 0.134145 * x * x)
        return x * (1 + t) / 2, d, torch.full_like(x, 1.0)
    if kind == "sigmoid":
        s = _sigmoid(x)
        return s, s * (1 - s), torch.full_like(x, 0.1)
    if kind == "tanh":
        t = torch.tanh(x)
        return t, 1 - t * t, torch.full_like(x, 0.8)
    if kind == "softplus":
        return torch.nn.functional.softplus(x, threshold=1e9), _sigmoid(x), torch.full_like(x, 0.25)
    assert kind == "situ"
    t, s = torch.tanh(x / 4), _sigmoid(x)
    return 4 * t * s, (1 - t * t) * s + 4 * t * s * (1 - s), torch.full_like(x, 1.0)


def act(kind, z, dtype):
    """(a(z), a'(z)) of a V: the first within |a'| e + 0.5 |a''| e^2 (the slope's own change by
    |a''| e), and 16 operations' roundings."""
    if kind is None:
        return z, V(torch.ones_like(z.v))
    a, d, dd = activation(kind, z.v, dtype)
    own = 16 * U * (1 + z.v.abs() + a.abs() + d.abs())
    own_d = 16 * U * (1 + z.v.abs()) ** 2
    return V(a, (d.abs() + dd * z.e) * z.e + own), V(d, dd * z.e + own_d)


def times(a, b):
    v = a.v * b.v
    e = a.e * (b.v.abs() + b.e) + a.v.abs() * b.e
    return V(v, e + 4 * U * (v.abs() + e))


def clip_up(ffn, u):
    """(cap(clip(u)), its derivative) of a V. Values within their error of a limit have either
    side's derivative."""
    d = V(torch.ones_like(u.v))
    if ffn.limit is not None:
        near = ((u.v.abs() - ffn.limit).abs() <= u.e)
        inside = (u.v.abs() < ffn.limit).to(F64)
        inside = torch.where(u.v.abs() == ffn.limit, 0.5, inside)
        d = V(inside, torch.where(near & (u.e > 0), 1.0, 0.0))
        u = V(u.v.clamp(-ffn.limit, ffn.limit), u.e)
    if ffn.up_softcap is not None:
        c = ffn.up_softcap
        t = torch.tanh(u.v / c)
        d = times(d, V(1 - t * t, u.e / c + 16 * U * (1 + u.v.abs() / c)))
        u = V(c * t, u.e + 16 * U * (c + u.v.abs()))
    return u, d


def units(ffn, z, gated, dtype):
    """(h, dh/du, dh/dg) of z (m, f, p)."""
    u, du = clip_up(ffn, V(z.v[..., 0], z.e[..., 0]))
    if not gated:
        a, s = act(ffn.activation, u, dtype)
        return a, times(s, du), None
    g = V(z.v[..., 1], z.e[..., 1])
    below = V(torch.ones_like(g.v))
    if ffn.limit is not None:
        near = (g.v - ffn.limit).abs() <= g.e
        w = torch.where(g.v == ffn.limit, 0.5, (g.v < ffn.limit).to(F64))
        below = V(w, torch.where(near & (g.e > 0), 1.0, 0.0))
        g = V(g.v.clamp(max=ffn.limit), g.e)
    a, s = act(ffn.activation, g, dtype)
    uo = V(u.v + ffn.up_offset, u.e + 2 * U * (u.v.abs() + abs(ffn.up_offset)))
    return times(a, uo), times(a, du), times(times(uo, s), below)


def kept(saved):
    """The projections that the backward works from: bfloat16 with their next 8 bits, where kept."""
    if saved.low is None:
        return saved.projected.to(F64)
    bits = (saved.projected.contiguous().view(torch.int16).to(torch.int32) << 16) + (
        saved.low.to(torch.int32) << 8)
    return bits.view(torch.float32).to(F64)


def randn(g, *shape, scale=1.0):
    return scale * torch.randn(*shape, generator=g, dtype=F64)
