"""The dense feed-forward block (bux_amd.mlp) against its formula in float64, within bounds
counted beforehand (tests/_dense.py): the forward from its inputs, the backward from what the
forward kept."""

import pytest
import torch

from _dense import BF16, F32, F64, V, kept, randn, times, units
from _util import announce

pytestmark = pytest.mark.gpu

# m, d, f: one token, odd everything, tiles' edges, few rows of long sums, whole tiles, no rows
SHAPES = [(1, 8, 4), (1, 2048, 96), (3, 7, 5), (33, 130, 67), (129, 257, 65), (200, 96, 264),
          (256, 512, 256), (520, 264, 392), (16, 4104, 72), (0, 32, 16)]


def _settings():
    from bux_amd.moe import Ffn

    return {"swish": Ffn(), "clamped": Ffn("swish", 1.5, 1.0), "capped": Ffn("gelu", None, 0.0, 2.0),
            "quick": Ffn("quick_gelu", 2.0, 1.0, 3.0), "relu2": Ffn("relu2"), "situ": Ffn("situ")}


def _make(g, dtype, m, d, f, p):
    s = {"x": randn(g, m, d), "up": randn(g, d, f, p, scale=d ** -0.5),
         "down": randn(g, f, d, scale=f ** -0.5), "up_bias": randn(g, f, p, scale=0.5),
         "down_bias": randn(g, d, scale=0.5), "residual": randn(g, m, d),
         "dy": randn(g, m, d, scale=0.1)}
    return {k: v.to(dtype).cuda() for k, v in s.items()}


def _v(t):
    return V(t.cpu().to(F64))


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("p", [2, 1], ids=["gated", "plain"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(lib, shape, p, dtype):
    from bux_amd import mlp

    m, d, f = shape
    g = torch.Generator().manual_seed(m + 3 * d + 5 * f + p)
    t = _make(g, dtype, m, d, f, p)
    for name, ffn in _settings().items():
        biased = name in ("clamped", "quick")
        ub, db = (t["up_bias"], t["down_bias"]) if biased else (None, None)
        res = t["residual"] if name in ("clamped", "relu2") else None
        announce("mlp", shape, p, dtype, name)
        r = mlp.feed_forward(t["x"], t["up"], t["down"], ffn, ub, db, res)
        z = _v(t["x"]) @ V(_v(t["up"]).v.view(d, f * p))
        if biased:
            z = z + V(_v(ub).v.view(-1))
        zp = V(z.v.view(m, f, p), z.e.view(m, f, p))
        zp.rounded(dtype).holds(r.saved.projected, "projected")
        assert (r.saved.low is None) == (dtype == F32)
        if dtype == BF16:  # in units of 2^8 of a 23-bit mantissa, one more where a byte ends
            V(zp.v, zp.e + 2.0 ** -15 * (zp.v.abs() + zp.e)).holds(kept(r.saved), "24 bits")
        h = units(ffn, zp, p == 2, dtype)[0].rounded(dtype)
        h.holds(r.saved.h, "h")
        y = _v(r.saved.h) @ _v(t["down"])
        if biased:
            y = y + _v(db)
        if res is not None:
            y = y + _v(res)
        y.rounded(dtype).holds(r.out, "out")
        bare = mlp.feed_forward(t["x"], t["up"], t["down"], ffn, ub, db, res, keep=False)
        assert bare.saved is None and torch.equal(bare.out, r.out)

        got = mlp.feed_forward_backward(t["dy"], r.saved, t["up"], t["down"], ffn, bias=biased)
        dh = _v(t["dy"]) @ _v(t["down"]).t()
        _, du, dg = units(ffn, _v(kept(r.saved)), p == 2, dtype)
        parts = [times(dh, s) for s in (du, dg)[:p]]
        exact = V(torch.stack([q.v for q in parts], -1).view(m, f * p),
                  torch.stack([q.e for q in parts], -1).view(m, f * p))
        dp = exact.rounded(dtype)
        up = V(_v(t["up"]).v.view(d, f * p))
        (dp @ up.t()).rounded(dtype).holds(got.x, "dx")
        dup = (_v(t["x"]).t() @ dp).rounded(dtype)
        V(dup.v.view(d, f, p), dup.e.view(d, f, p)).holds(got.up, "dup")
        (_v(r.saved.h).t() @ _v(t["dy"])).rounded(dtype).holds(got.down, "ddown")
        if biased:
            # its 24 bits (of bfloat16), not the 16 that the products take
            low = 2.0 ** -15 * (exact.v.abs() + exact.e) if dtype == BF16 else 0.0
            s = V(exact.v, exact.e + low).sum0().rounded(dtype)
            V(s.v.view(f, p), s.e.view(f, p)).holds(got.up_bias, "dup_bias")
            _v(t["dy"]).sum0().rounded(dtype).holds(got.down_bias, "ddown_bias")
        else:
            assert got.up_bias is None and got.down_bias is None


@pytest.mark.parametrize("m", [5, 200])
def test_backward_from_the_bfloat16_projections_alone(lib, m):
    from bux_amd import mlp
    from bux_amd.moe import Ffn

    g = torch.Generator().manual_seed(m)
    d, f = 136, 72
    t = _make(g, BF16, m, d, f, 2)
    r = mlp.feed_forward(t["x"], t["up"], t["down"])
    alone = r.saved._replace(low=None)
    announce("mlp without low bytes", m)
    got = mlp.feed_forward_backward(t["dy"], alone, t["up"], t["down"])
    dh = _v(t["dy"]) @ _v(t["down"]).t()
    _, du, dg = units(Ffn(), _v(kept(alone)), True, BF16)
    parts = [times(dh, s) for s in (du, dg)]
    dp = V(torch.stack([q.v for q in parts], -1).view(m, f * 2),
           torch.stack([q.e for q in parts], -1).view(m, f * 2)).rounded(BF16)
    (dp @ V(_v(t["up"]).v.view(d, f * 2)).t()).rounded(BF16).holds(got.x, "dx")


def test_projections_at_the_ends_of_their_type(lib):
    """Values that round to infinity, infinities, NaN, zeros and the smallest, through the kept 24
    bits: h is act(u) of a plain relu block with one input a unit, dp its gradient."""
    from bux_amd import mlp
    from bux_amd.moe import Ffn

    vals = [3.3e38, -3.3e38, float("inf"), float("-inf"), float("nan"), 0.0, -0.0, 1e-38, 1.0, -1.0,
            2.0 ** -126, 255.5]
    up = torch.tensor(vals, dtype=BF16, device="cuda").view(1, -1, 1).contiguous()
    f = len(vals)
    x = torch.tensor([[1.0], [1.00390625 * 1.0]], dtype=BF16, device="cuda")
    down = torch.ones(f, 1, dtype=BF16, device="cuda")
    announce("mlp ends of bfloat16")
    r = mlp.feed_forward(x, up, down, Ffn("relu"))
    v = up.view(-1).double()
    want = kept(r.saved)[0, :, 0]
    assert torch.equal(want.isnan(), v.isnan())
    assert torch.equal(want[~v.isnan()], v[~v.isnan()])
    got = mlp.feed_forward_backward(torch.ones_like(x), r.saved, up, down, Ffn("relu"))
    # d up = x^T dp with dp = 1 where the projection is above 0, 0 where it is not
    sums = x.double().sum().item()
    for j, val in enumerate(vals):
        if val == val:
            assert abs(got.up.view(-1)[j].item() - (sums if val > 0 else 0.0)) <= 2.0 ** -8 * sums


def test_gradients_against_differences(lib):
    """float32, along a random direction of every input, against a central difference of the
    formula in float64."""
    from bux_amd import mlp
    from bux_amd.moe import Ffn

    g = torch.Generator().manual_seed(21)
    m, d, f = 19, 33, 27
    t = _make(g, F32, m, d, f, 2)
    ffn = Ffn("swish", None, 1.0)
    r = mlp.feed_forward(t["x"], t["up"], t["down"], ffn, t["up_bias"], t["down_bias"])
    got = mlp.feed_forward_backward(t["dy"], r.saved, t["up"], t["down"], ffn, bias=True)
    names = ("x", "up", "down", "up_bias", "down_bias")
    v = {n: randn(g, *t[n].shape) for n in names}

    def loss(e):
        q = {n: t[n].cpu().to(F64) + e * v[n] for n in names}
        z = q["x"] @ q["up"].reshape(d, f * 2) + q["up_bias"].view(-1)
        z = z.view(m, f, 2)
        h = z[..., 1] * torch.sigmoid(z[..., 1]) * (z[..., 0] + 1)
        return (t["dy"].cpu().to(F64) * (h @ q["down"] + q["down_bias"])).sum()

    want = (loss(1e-4) - loss(-1e-4)) / 2e-4
    grads = dict(zip(names, (got.x, got.up, got.down, got.up_bias, got.down_bias)))
    parts = [grads[n].cpu().to(F64) * v[n] for n in names]
    scale = sum(q.abs().sum() for q in parts)
    # under 200 roundings of float32 each, and the difference's own 1e-8 times the third derivative
    assert abs(sum(q.sum() for q in parts) - want) <= (400 * 2.0 ** -24 + 1e-6) * scale


def test_a_captured_step_replays_as_the_eager_one(lib):
    from bux_amd import mlp

    g = torch.Generator().manual_seed(30)
    m, d, f = 300, 264, 200
    static = _make(g, BF16, m, d, f, 2)

    def step(t):
        r = mlp.feed_forward(t["x"], t["up"], t["down"], up_bias=t["up_bias"],
                             down_bias=t["down_bias"], residual=t["residual"])
        b = mlp.feed_forward_backward(t["dy"], r.saved, t["up"], t["down"], bias=True)
        return [r.out, *b]

    announce("mlp graph")
    step(static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(static)
    for replay in range(3):
        fresh = _make(g, BF16, m, d, f, 2)
        for k in static:
            static[k].copy_(fresh[k])
        torch.cuda.synchronize()
        announce("mlp graph replay", replay)
        graph.replay()
        torch.cuda.synchronize()
        want = step(fresh)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))


def test_a_layer_of_experts_and_a_shared_one(lib):
    """A layer as a model runs it: the tokens' norm, the routed experts and the dense block beside
    them onto one residual stream, back through both, and every gradient clipped together."""
    from bux_amd import clip, mlp, moe, norm, router

    g = torch.Generator().manual_seed(40)
    t, d, f, e, k = 96, 256, 128, 8, 2
    x = randn(g, t, d).to(BF16).cuda()
    gain = (1 + 0.1 * randn(g, d)).to(BF16).cuda()
    kernel = randn(g, d, e, scale=0.1).to(BF16).cuda()
    up, down = (randn(g, e, d, f, 2, scale=0.05).to(BF16).cuda(),
                randn(g, e, f, d, scale=0.05).to(BF16).cuda())
    sup, sdown = (randn(g, d, f, 2, scale=0.05).to(BF16).cuda(),
                  randn(g, f, d, scale=0.05).to(BF16).cuda())
    announce("layer with a shared expert")
    n = norm.normed(x, moe.ExpertNorm(), gain)
    r = router.route(n.out, kernel, top_k=k, with_logits=True)
    y, saved = moe.experts_forward(n.out, r.idx, r.weights, up, down, fmt="compute")
    s = mlp.feed_forward(n.out, sup, sdown, residual=y)
    # the block onto the experts' output: their sum, rounded once
    alone = mlp.feed_forward(n.out, sup, sdown)
    hv = V(alone.saved.h.cpu().to(F64)) @ V(sdown.cpu().to(F64)) + V(y.cpu().to(F64))
    hv.rounded(BF16).holds(s.out, "block onto experts")

    dy = randn(g, t, d, scale=0.1).to(BF16).cuda()
    ge = moe.experts_backward(saved, dy, up, down, fmt="compute")
    gs = mlp.feed_forward_backward(dy, s.saved, sup, sdown)
    gr = router.route_backward(n.out, kernel, r.idx, r.logits, ge["weights"], dz=ge["z"])
    gn = norm.normed_backward(gr.x + gs.x, x, n.stats, moe.ExpertNorm(), gain)
    grads = [ge["up"], ge["down"], gs.up, gs.down, gr.kernel, gn.scale]
    c = clip.clipped(grads, 0.5)
    want = sum(q.cpu().to(F64).square().sum() for q in grads).sqrt()
    assert abs(c.norm.item() - want) <= 2.0 ** -22 * want and want > 0.5
    for q, o in zip(grads, c.grads):
        V(q.cpu().to(F64) * (0.5 / want), 4 * 2.0 ** -24 * q.cpu().to(F64).abs()
          ).rounded(q.dtype).holds(o, "clipped")


def test_refusals(lib):
    from bux_amd import mlp

    x = torch.zeros(4, 32, dtype=BF16, device="cuda")
    up = torch.zeros(32, 16, 2, dtype=BF16, device="cuda")
    down = torch.zeros(16, 32, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="up is"):
        mlp.feed_forward(x, up.view(32, 32), down)
    with pytest.raises(ValueError, match="up is"):
        mlp.feed_forward(x, up.view(32, 8, 4), down)
    with pytest.raises(ValueError, match="down"):
        mlp.feed_forward(x, up, down[:8])
    with pytest.raises(ValueError, match="rows of 32"):
        mlp.feed_forward(x[:, :8].contiguous(), up, down)
    with pytest.raises(TypeError, match="float32"):
        mlp.feed_forward(x, up.float(), down)
    with pytest.raises(ValueError, match="up_bias"):
        mlp.feed_forward(x, up, down, up_bias=x[0])
    with pytest.raises(ValueError, match="down_bias"):
        mlp.feed_forward(x, up, down, down_bias=x)
    with pytest.raises(ValueError, match="residual"):
        mlp.feed_forward(x, up, down, residual=x[:2])
    r = mlp.feed_forward(x, up, down)
    with pytest.raises(ValueError, match="dy"):
        mlp.feed_forward_backward(x[:2], r.saved, up, down)
    with pytest.raises(ValueError, match="projected"):
        mlp.feed_forward_backward(x, r.saved._replace(projected=r.saved.h), up, down)
    with pytest.raises(ValueError, match="h is"):
        mlp.feed_forward_backward(x, r.saved._replace(h=x), up, down)
    with pytest.raises(ValueError, match="low is"):
        mlp.feed_forward_backward(x, r.saved._replace(low=r.saved.low[..., 0].contiguous()), up, down)
    with pytest.raises(ValueError, match="low is int8"):
        mlp.feed_forward_backward(x, r.saved._replace(low=r.saved.low.float()), up, down)
