"""The tokens' norm (bux_amd.norm) against its formula in float64.

Tolerances count roundings: one to the outputs' type (half a step, eps / 2 of the value), and
float32's inside (u = 2^-24 each). A row's sums pass at most 24 values a lane, 6 exchanges and
8 waves: 40 additions, and a handful of products and a division follow, so that DEPTH = 64
roundings bound each sum's and each factor's error relative to the magnitudes that go in.
"""

import ctypes

import pytest
import torch

from _util import announce
from bux_amd import _lib
from bux_amd.moe import ExpertNorm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DEPTH = 64
BF16, F32 = torch.bfloat16, torch.float32

# one row and many, a turn more than the backward's workgroups hold, one chunk and all, each
# count of waves, rows of no whole eights, the widest
SIZES = [(1, 8), (3, 9), (1, 2048), (5, 1443), (7, 1536), (2, 1537), (130, 2880), (33, 3001),
         (4, 6144), (3, 6145), (2, 12281), (3, 12288), (2100, 64), (4500, 17), (0, 64)]

SETTINGS = {
    "rms": ExpertNorm("rmsnorm"),
    "rms bare": ExpertNorm("rmsnorm", affine=False),
    "rms zero-centered": ExpertNorm("rmsnorm", 1e-5, zero_centered=True),
    "rms scale input": ExpertNorm("rmsnorm", scale_input=True),
    "layer": ExpertNorm("layernorm", 1e-5, bias=True),
    "layer bare with bias": ExpertNorm("layernorm", affine=False, bias=True),
    "layer zero-centered scale input": ExpertNorm("layernorm", bias=True, zero_centered=True,
                                                  scale_input=True),
}


def _inputs(m, d, dtype, norm, seed=0):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, dtype=torch.float64)

    x = normal(m, d) + 0.5 * normal(d)
    if x.numel():
        x.view(-1)[torch.randint(x.numel(), (max(1, x.numel() // 500),), generator=g)] *= 50
    t = {"x": x, "residual": normal(m, d), "dy": normal(m, d), "d_summed": normal(m, d),
         "scale": 1 + 0.2 * normal(d) if not norm.zero_centered else 0.2 * normal(d),
         "bias": 0.3 * normal(d)}
    return {k: v.to(dtype).cuda() for k, v in t.items()}


def _parameters(norm, t):
    return t["scale"] if norm.affine else None, t["bias"] if norm.bias else None


def _formula(x, norm, scale, bias):
    """(out, c, r, gain, |v|'s mean) of float64 rows."""
    gain = x.new_ones(x.shape[1])
    if norm.affine:
        gain = scale.double() + (1.0 if norm.zero_centered else 0.0)
    v = x * gain if norm.affine and norm.scale_input else x
    c = v - v.mean(-1, keepdim=True) if norm.kind == "layernorm" else v
    r = 1 / (c.square().mean(-1, keepdim=True) + norm.eps).sqrt()
    out = c * r
    if norm.affine and not norm.scale_input:
        out = out * gain
    if norm.bias:
        out = out + bias.double()
    return out, c, r, gain, v.abs().mean(-1, keepdim=True)


def _check(got, want, tolerance, what):
    got = got.double()
    assert got.shape == want.shape
    off = (got - want).abs() / tolerance
    assert not torch.isnan(got).any(), what
    assert off.numel() == 0 or off.max() <= 1, (what, float(off.max()))


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("name", list(SETTINGS))
@pytest.mark.parametrize("m,d", SIZES)
def test_forward_and_backward(lib, m, d, name, dtype):
    from bux_amd import norm as tnorm
    norm = SETTINGS[name]
    announce("norm", m, d, name, dtype)
    t = _inputs(m, d, dtype, norm)
    scale, bias = _parameters(norm, t)
    eps = torch.finfo(dtype).eps
    for residual in (None, t["residual"]):
        r = tnorm.normed(t["x"], norm, scale, bias, residual=residual)
        x = t["x"]
        if residual is None:
            assert r.summed is None
        else:
            x = (t["x"].float() + residual.float()).to(dtype)
            assert torch.equal(r.summed, x)
        out, c, rstd, gain, size = _formula(x.double(), norm, scale, bias)
        g = gain.abs() if norm.affine and not norm.scale_input else torch.ones_like(gain)
        inside = DEPTH * U * (rstd * (c.abs() + size) * g + (bias.double().abs() if norm.bias else 0))
        _check(r.out, out, eps / 2 * out.abs() + inside + 1e-30, "out")

        past = None if residual is None else t["d_summed"]
        grads = tnorm.normed_backward(t["dy"], x, r.stats, norm, scale, past)
        dy = t["dy"].double()
        inner = norm.affine and not norm.scale_input
        h = dy * gain if inner else dy
        n = c * rstd
        far = n.abs() + rstd * size  # what n's roundings are relative to
        mean = (lambda v: v.mean(-1, keepdim=True))
        dv = rstd * (h - n * mean(h * n) - (mean(h) if norm.kind == "layernorm" else 0))
        off = 3 * DEPTH * U * rstd * (h.abs() + mean(h.abs()) + far * mean(h.abs() * far))
        dx = dv
        if norm.affine and norm.scale_input:
            dx, outer = dv * gain, off * gain.abs()
        else:
            outer = off
        if past is not None:
            dx = dx + past.double()
            outer = outer + 2 * U * past.double().abs()
        _check(grads.x, dx, eps / 2 * dx.abs() + outer + 1e-30, "dx")
        rows = (m + DEPTH) * U  # a column's sum: at most a rounding a row
        if norm.affine:
            if norm.scale_input:
                want, tol = (dv * x.double()).sum(0), ((off + rows * dv.abs()) * x.double().abs()).sum(0)
            else:
                want, tol = (dy * n).sum(0), (rows + 3 * DEPTH * U) * (dy.abs() * far).sum(0)
            assert grads.scale.dtype == F32
            _check(grads.scale, want, tol + 1e-30, "scale")
        else:
            assert grads.scale is None
        if norm.bias:
            assert grads.bias.dtype == F32
            _check(grads.bias, dy.sum(0), rows * dy.abs().sum(0) + 1e-30, "bias")
        else:
            assert grads.bias is None


@pytest.mark.parametrize("name", ["rms", "layer", "layer zero-centered scale input"])
def test_gradients_against_differences(lib, name):
    """The formula's central differences along random directions, in float64, and the
    gradients that the op gives in float32: the differences' own error is of step^2."""
    from bux_amd import norm as tnorm
    norm = SETTINGS[name]
    m, d = 6, 300
    t = _inputs(m, d, F32, norm, seed=3)
    scale, bias = _parameters(norm, t)
    x = t["x"]
    r = tnorm.normed(x, norm, scale, bias)
    grads = tnorm.normed_backward(t["dy"], x, r.stats, norm, scale)
    dy, step = t["dy"].double(), 1e-5
    g = torch.Generator().manual_seed(9)

    def loss(x, scale, bias):
        return float((dy * _formula(x, norm, scale, bias)[0]).sum())

    for which, grad in (("x", grads.x), ("scale", grads.scale), ("bias", grads.bias)):
        if grad is None:
            continue
        at = {"x": x.double(), "scale": scale.double(), "bias": None if bias is None else bias.double()}
        v = torch.randn(at[which].shape, generator=g, dtype=torch.float64).cuda()
        up, down = dict(at), dict(at)
        up[which], down[which] = at[which] + step * v, at[which] - step * v
        want = (loss(**up) - loss(**down)) / (2 * step)
        got = float((grad.double() * v).sum())
        # float32 gradients: DEPTH roundings of each term's magnitude; the differences: the
        # losses' float64 cancellation over the step and the step's square
        size = float((grad.double() * v).abs().sum())
        assert abs(got - want) <= 3 * DEPTH * U * size + 1e-6 * abs(want) + 1e-5, (which, got, want)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_rows_at_any_element_and_nothing_past_the_rows(lib, dtype):
    """Rows that begin at an odd element (a slice's), and buffers whose other elements stay."""
    m, d = 5, 1001
    norm = SETTINGS["layer"]
    t = _inputs(m, d, dtype, norm, seed=5)
    st = norm.struct()

    def inside(v=None):
        buf = torch.full((m * d + 64,), 7.0, dtype=dtype, device="cuda")
        at = buf[3:3 + m * d].view(m, d)
        if v is not None:
            at.copy_(v)
        return buf, at

    bufs = {k: inside(t[k]) for k in ("x", "residual", "dy", "d_summed")}
    out_buf, out = inside()
    sum_buf, summed = inside()
    dx_buf, dx = inside()
    stats = torch.full((m + 1, 2), 7.0, device="cuda")
    params = torch.full((2, d + 1), 7.0, device="cuda")
    ws = torch.empty(lib.bux_norm_backward_workspace_size(m, d), dtype=torch.uint8, device="cuda")
    forward = lib.bux_norm_forward if dtype == BF16 else lib.bux_norm_forward_f32
    backward = lib.bux_norm_backward if dtype == BF16 else lib.bux_norm_backward_f32
    p = (lambda v: v.data_ptr())
    _lib.check(forward(p(bufs["x"][1]), p(bufs["residual"][1]), m, d, ctypes.byref(st), p(t["scale"]),
                       p(t["bias"]), p(summed), p(out), p(stats), None))
    _lib.check(backward(p(bufs["dy"][1]), p(summed), p(stats), p(bufs["d_summed"][1]), m, d,
                        ctypes.byref(st), p(t["scale"]), p(dx), p(params[0]), p(params[1]), p(ws),
                        ws.numel(), None))
    from bux_amd import norm as tnorm
    r = tnorm.normed(t["x"], norm, t["scale"], t["bias"], residual=t["residual"])
    g = tnorm.normed_backward(t["dy"], r.summed, r.stats, norm, t["scale"], t["d_summed"])
    assert torch.equal(out, r.out) and torch.equal(summed, r.summed) and torch.equal(dx, g.x)
    assert torch.equal(stats[:m], r.stats)
    assert torch.equal(params[0, :d], g.scale) and torch.equal(params[1, :d], g.bias)
    for buf in (out_buf, sum_buf, dx_buf):
        assert (buf[:3] == 7).all() and (buf[3 + m * d:] == 7).all()
    assert (stats[m] == 7).all() and (params[:, d] == 7).all()


@pytest.mark.parametrize("m,d", [(1, 64), (3, 7168), (9, 512), (700, 2880), (1100, 4096), (2100, 1024)])
def test_the_same_bits_at_any_alignment(lib, m, d):
    """Aligned rows pass LDS a row ahead, rows an element off load in their turn: the same sums."""
    from bux_amd import norm as tnorm
    from bux_amd.moe import ExpertNorm
    announce("norm alignment", m, d)
    norm = ExpertNorm("layernorm", bias=True)
    t = _inputs(m, d, BF16, norm, seed=m)
    off = {}
    for k, v in t.items():
        buffer = torch.zeros(v.numel() + 1, dtype=v.dtype, device="cuda")
        off[k] = buffer[1:].view(v.shape).copy_(v)
    got = []
    for v in (t, off):
        f = tnorm.normed(v["x"], norm, v["scale"], v["bias"])
        g = tnorm.normed_backward(v["dy"], v["x"], f.stats, norm, v["scale"], d_summed=v["d_summed"])
        got.append((f.out, f.stats, *g))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_rows_of_nan_and_infinity_stay_their_own(lib):
    """A row that holds a NaN or an infinity is not a number; the rows beside it, in its own
    workgroup too, are what they are without it."""
    from bux_amd import norm as tnorm
    for m, d in ((9, 64), (9, 1601), (5, 5000)):
        norm = SETTINGS["layer"]
        t = _inputs(m, d, BF16, norm, seed=6)
        x = t["x"].clone()
        x[2, d - 1], x[4, 0] = float("nan"), float("inf")
        clean = tnorm.normed(t["x"], norm, t["scale"], t["bias"])
        r = tnorm.normed(x, norm, t["scale"], t["bias"])
        a = tnorm.normed_backward(t["dy"], t["x"], clean.stats, norm, t["scale"])
        b = tnorm.normed_backward(t["dy"], x, r.stats, norm, t["scale"])
        rest = [i for i in range(m) if i not in (2, 4)]
        assert torch.isnan(r.out[2]).all() and torch.isnan(r.out[4]).any()
        assert torch.equal(r.out[rest], clean.out[rest]) and torch.equal(a.x[rest], b.x[rest])
        assert torch.equal(a.bias, b.bias)


def test_a_row_of_zeros_and_one_of_equal_values(lib):
    from bux_amd import norm as tnorm
    d = 96
    x = torch.zeros(2, d, device="cuda")
    x[1] = 3.0
    norm = ExpertNorm("layernorm", 1e-6, affine=False)
    r = tnorm.normed(x, norm)
    assert (r.out == 0).all()
    assert torch.allclose(r.stats[:, 1], torch.full((2,), 1e3, device="cuda"), rtol=1e-6)
    r = tnorm.normed(x, ExpertNorm("rmsnorm", 1e-6, affine=False))
    assert (r.out[0] == 0).all() and torch.allclose(r.out[1], torch.ones(d, device="cuda"), rtol=1e-6)


def test_leading_dimensions_repeats_and_streams(lib):
    """(b, s, d) rows; the same bits each time, on another stream too."""
    from bux_amd import norm as tnorm
    norm = SETTINGS["layer"]
    t = _inputs(600, 770, BF16, norm, seed=7)
    r = tnorm.normed(t["x"], norm, t["scale"], t["bias"], residual=t["residual"])
    g = tnorm.normed_backward(t["dy"], r.summed, r.stats, norm, t["scale"], t["d_summed"])
    cube = (lambda v: v.view(4, 150, 770))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r2 = tnorm.normed(cube(t["x"]), norm, t["scale"], t["bias"], residual=cube(t["residual"]))
        g2 = tnorm.normed_backward(cube(t["dy"]), r2.summed, r2.stats, norm, t["scale"],
                                   cube(t["d_summed"]))
    torch.cuda.current_stream().wait_stream(side)
    assert r2.out.shape == (4, 150, 770)
    assert torch.equal(cube(r.out), r2.out) and torch.equal(cube(g.x), g2.x)
    assert torch.equal(g.scale, g2.scale) and torch.equal(g.bias, g2.bias)


def test_in_a_graph(lib):
    """Captured once, replayed over new inputs, with eager work between the replays."""
    from bux_amd import norm as tnorm
    norm = SETTINGS["layer"]
    t = _inputs(300, 1030, BF16, norm, seed=8)

    def step():
        r = tnorm.normed(t["x"], norm, t["scale"], t["bias"], residual=t["residual"])
        return r, tnorm.normed_backward(t["dy"], r.summed, r.stats, norm, t["scale"], t["d_summed"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, g = step()
    for seed in (10, 11, 12):
        for k, v in _inputs(300, 1030, BF16, norm, seed=seed).items():
            t[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        r2, g2 = step()
        torch.cuda.synchronize()
        assert torch.equal(r.out, r2.out) and torch.equal(r.summed, r2.summed)
        assert torch.equal(g.x, g2.x) and torch.equal(g.scale, g2.scale) and torch.equal(g.bias, g2.bias)


def test_refusals(lib):
    from bux_amd import norm as tnorm
    x = torch.zeros(4, 64, dtype=BF16, device="cuda")
    s = torch.zeros(64, dtype=BF16, device="cuda")
    norm = ExpertNorm("rmsnorm")
    with pytest.raises(ValueError, match="scale"):
        tnorm.normed(x, norm)
    with pytest.raises(TypeError, match="scale"):
        tnorm.normed(x, norm, s.float())
    with pytest.raises(ValueError, match="scale"):
        tnorm.normed(x, norm, s[:32])
    with pytest.raises(TypeError, match="float16"):
        tnorm.normed(x.half(), norm, s)
    with pytest.raises(ValueError, match="8 to 12288"):
        tnorm.normed(x[:, :7].contiguous(), norm, s)
    with pytest.raises(ValueError, match="residual"):
        tnorm.normed(x, norm, s, residual=x[:3])
    with pytest.raises(ValueError, match="contiguous"):
        tnorm.normed(x.t(), norm, s)
    with pytest.raises(ValueError, match="GPU"):
        tnorm.normed(x.cpu(), norm, s)
    with pytest.raises(ValueError, match="stats"):
        tnorm.normed_backward(x, x, torch.zeros(3, 2, device="cuda"), norm, s)
    with pytest.raises(ValueError, match="no norm"):
        tnorm.normed(x, ExpertNorm("batchnorm"), s)
