"""The router's backward (router.route_backward) against autograd of its formula in float64.

Tolerances count roundings (u = 2^-24): a logit's gradient G passes sums of at most 16 values a
lane and 6 exchanges and some dozens of products, divisions and exponentials (each within 2
units): DEPTH = 64 of u, relative to the magnitudes that go in. Its products take it in two
bfloat16 parts: 2^-17 of it. A sum over n logits or t tokens adds a rounding a term at most,
relative to the terms' magnitudes; the outputs' one rounding is half a bfloat16 step, 2^-8.
"""

import pytest
import torch

from _util import announce
from bux_amd import _lib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DEPTH = 64
PARTS = 2.0 ** -17
HALF_STEP = 2.0 ** -8
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def _inputs(t, d, n, scored, k, seed, spread=1.0, offset=0.0, sinks=False, scores=False,
            logits=False, dz=False):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, dtype=F64)

    z = (normal(t, n) * spread + offset).float()
    idx = (torch.topk(z[:, :scored], k, -1).indices.int() if t else torch.zeros(0, k).int())
    v = {"x": normal(t, d).to(BF16), "kernel": (0.1 * normal(d, n)).to(BF16), "idx": idx,
         "logits": z, "d_weights": normal(t, k).to(BF16),
         "d_sinks": normal(t, n - scored).to(BF16) if sinks else None,
         "d_scores": (0.1 * normal(t, scored)).float() if scores else None,
         "d_logits": (0.01 * normal(t, n)).float() if logits else None,
         "dz": normal(t, d).to(BF16) if dz else None}
    return {a: b if b is None else b.cuda() for a, b in v.items()}


def _scores(z, router):
    if router == "softmax":
        return torch.softmax(z, -1)
    if router == "sigmoid":  # as exp(-log(1 + e^-z)): its derivative s(-z) s(z) does not cancel
        return torch.exp(-torch.logaddexp(-z, torch.zeros_like(z)))
    return torch.sqrt(torch.logaddexp(z, torch.zeros_like(z)))


def _loss(z, v, scored, router, normalize, factor):
    """The loss whose gradient route_backward gives, as a function of the logits (float64)."""
    s = _scores(z, router)
    w = s.gather(1, v["idx"].long())
    sink = s[:, scored:]
    if normalize:
        total = w.sum(-1, keepdim=True) + sink.sum(-1, keepdim=True)
        w, sink = w / total, sink / total
    loss = (w * factor * v["d_weights"].double()).sum()
    if v["d_sinks"] is not None:
        loss = loss + (sink * factor * v["d_sinks"].double()).sum()
    if v["d_scores"] is not None:
        loss = loss + (s[:, :scored] * v["d_scores"].double()).sum()
    if v["d_logits"] is not None:
        loss = loss + (z * v["d_logits"].double()).sum()
    return loss


def _magnitude(v, scored, router, normalize, factor):
    """What G's roundings are relative to, a logit each."""
    z = v["logits"].double()
    s = _scores(z, router)
    at = v["idx"].long()
    w = s.gather(1, at)
    g = v["d_weights"].double().abs() * factor
    gs = torch.zeros_like(s)
    if v["d_sinks"] is not None:
        gs[:, scored:] = v["d_sinks"].double().abs() * factor
    if normalize:
        total = w.sum(-1, keepdim=True) + s[:, scored:].sum(-1, keepdim=True)
        shift = ((g * w).sum(-1, keepdim=True) + (gs * s).sum(-1, keepdim=True)) / total
        g, gs[:, scored:] = (g + shift) / total, (gs[:, scored:] + shift) / total
    ds = gs.scatter_add(1, at, g)
    if v["d_scores"] is not None:
        ds[:, :scored] += v["d_scores"].double().abs()
    if router == "softmax":
        m = s * (ds + (ds * s).sum(-1, keepdim=True))
        # exp(z - max) has the argument's own rounding: |z - max| u of the score
        m = m * (1 + (z.max(-1, keepdim=True).values - z) / DEPTH)
    elif router == "sigmoid":
        m = ds * s * torch.sigmoid(-z)
    else:
        m = ds * torch.sigmoid(z) / (2 * s).clamp_min(1e-30)
    if v["d_logits"] is not None:
        m = m + v["d_logits"].double().abs()
    return m


def _check(got, want, tolerance, what):
    got = got.double()
    assert got.shape == want.shape and not torch.isnan(got).any(), what
    off = (got - want).abs() / (tolerance + 1e-30)
    assert off.numel() == 0 or off.max() <= 1, (what, float(off.max()))


def _run(v, scored, router, normalize, scale, scaling):
    from bux_amd import router as r
    return r.route_backward(
        v["x"], v["kernel"], v["idx"], v["logits"], v["d_weights"], scored=scored, router=router,
        router_logit_scale=scale, normalize_top_k=normalize, routed_scaling_factor=scaling,
        d_sinks=v["d_sinks"], d_scores=v["d_scores"], d_logits=v["d_logits"], dz=v["dz"])


def _compare(v, scored, router, normalize, scale, scaling):
    t, n = v["logits"].shape
    got = _run(v, scored, router, normalize, scale, scaling)
    factor = float(torch.tensor(scaling, dtype=BF16))
    z = v["logits"].double().requires_grad_()
    G = torch.autograd.grad(_loss(z, v, scored, router, normalize, factor), z)[0]
    off = DEPTH * U * (_magnitude(v, scored, router, normalize, factor) + G.abs())
    G, off = G * scale, off * abs(scale)
    x, kernel = v["x"].double(), v["kernel"].double()
    part = off + PARTS * G.abs()
    dx = G @ kernel.t().contiguous()
    tol = (part + n * U * G.abs()) @ kernel.abs().t().contiguous()
    if v["dz"] is not None:
        dx = dx + v["dz"].double()
        tol = tol + U * (v["dz"].double().abs() + dx.abs())
    _check(got.x, dx, HALF_STEP * dx.abs() + 2 * tol, "x")
    dk = x.t().contiguous() @ G
    tol = x.abs().t().contiguous() @ (part + t * U * G.abs())
    _check(got.kernel, dk, HALF_STEP * dk.abs() + 2 * tol, "kernel")
    _check(got.bias, G.sum(0), (off + t * U * G.abs()).sum(0), "bias")


CASES = [
    # t, d, n, scored, k, router, normalize, logit scale, scaling, and the extras
    (1, 16, 8, 8, 2, "softmax", True, 1.0, 1.0, {}),
    (1, 2048, 128, 128, 8, "softmax", True, 1.0, 1.0, {"dz": True}),
    (3, 48, 1, 1, 1, "sigmoid", True, 1.0, 1.0, {}),
    (33, 144, 31, 31, 4, "softmax", True, 0.5, 2.5, {"dz": True, "scores": True}),
    (65, 528, 60, 60, 6, "sigmoid", True, 1.0, 2.827, {"logits": True}),
    (500, 128, 130, 128, 8, "softmax", True, 1.0, 1.0, {"sinks": True, "scores": True}),
    (257, 272, 66, 64, 1, "sigmoid", False, 2.0, 1.0, {"sinks": True, "logits": True}),
    (129, 64, 32, 32, 16, "sqrtsoftplus", True, 1.0, 2.5, {"scores": True, "dz": True}),
    (700, 640, 256, 256, 8, "sigmoid", True, 1.0, 2.5, {"scores": True}),
    (40, 112, 1000, 1000, 16, "softmax", False, 1.0, 1.0, {"scores": True, "logits": True}),
    (70, 16, 1024, 1020, 3, "sqrtsoftplus", True, -1.0, 1.0, {"sinks": True}),
    (5, 96, 300, 290, 2, "softmax", True, 1.0, 1.0, {}),  # sinks without a gradient of their own
    (4100, 176, 40, 40, 4, "softmax", True, 1.0, 1.0, {"dz": True}),
    (0, 64, 40, 40, 4, "softmax", True, 1.0, 1.0, {"dz": True}),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}x{c[1]}x{c[2]}-{c[5]}")
def test_against_autograd(lib, case):
    t, d, n, scored, k, router, normalize, scale, scaling, extras = case
    announce("route backward", case)
    _compare(_inputs(t, d, n, scored, k, seed=t + n, **extras), scored, router, normalize, scale,
             scaling)


@pytest.mark.parametrize("router", ["softmax", "sigmoid", "sqrtsoftplus"])
@pytest.mark.parametrize("spread,offset", [(30.0, 0.0), (1.0, 60.0), (1.0, -60.0)])
def test_far_logits(lib, router, spread, offset):
    announce("route backward", router, spread, offset)
    # off the softmax, unnormalized: scores far below 1 would make the picks' sum the divisor
    v = _inputs(50, 64, 48, 48, 4, seed=5, spread=spread, offset=offset, scores=True)
    _compare(v, 48, router, router == "softmax", 1.0, 1.0)


def test_scores_that_underflow_have_no_gradient(lib):
    """sqrt(softplus) of a logit whose exponential is 0, and a sigmoid's: 0, not NaN."""
    for router in ("sqrtsoftplus", "sigmoid"):
        v = _inputs(4, 32, 16, 16, 2, seed=6, scores=True)
        v["logits"][:, 3:6] = -300.0
        v["logits"][1] = -300.0
        got = _run(v, 16, router, True, 1.0, 1.0)
        assert not torch.isnan(got.x).any() and not torch.isnan(got.kernel).any()
        assert (got.x[1] == 0).all() and (got.bias[3:6] == 0).all()


@pytest.mark.parametrize("router", ["softmax", "sigmoid", "sqrtsoftplus"])
def test_a_normalized_single_pick_is_constant(lib, router):
    """Its weight is 1 whatever the logits, so its gradient is 0 and no rounding's remainder."""
    v = _inputs(70, 64, 40, 40, 1, seed=8, dz=True)
    got = _run(v, 40, router, True, 2.5, 1.0)
    assert torch.equal(got.x, v["dz"])
    assert (got.kernel == 0).all() and (got.bias == 0).all()


@pytest.mark.parametrize("offset", [-80.0, -86.0, -95.0])
def test_picks_of_tiny_scores(lib, offset):
    """Normalized sigmoids about the smallest normal number: finite gradients."""
    v = _inputs(20, 32, 24, 24, 4, seed=9, offset=offset, scores=True)
    got = _run(v, 24, "sigmoid", True, 1.0, 1.0)
    for g in (got.x, got.kernel, got.bias):
        assert torch.isfinite(g).all()


def test_picks_made_twice_and_outside(lib):
    """A pick made twice counts twice in the sum; one outside the scored experts not at all."""
    v = _inputs(6, 64, 20, 18, 3, seed=7)
    v["idx"][0] = torch.tensor([4, 4, 2])
    _compare(v, 18, "softmax", True, 1.0, 1.0)
    w = {key: None if x is None else x.clone() for key, x in v.items()}
    w["idx"][1] = torch.tensor([18, -1, 5])
    w["idx"][2] = torch.tensor([2**31 - 1, -2**31, 19])
    got = _run(w, 18, "sigmoid", False, 1.0, 1.0)
    one = {key: None if x is None else x.clone() for key, x in w.items()}
    one["idx"][1], one["idx"][2] = torch.tensor([0, 0, 5]), torch.tensor([0, 0, 0])
    one["d_weights"][1, :2] = 0
    one["d_weights"][2] = 0
    want = _run(one, 18, "sigmoid", False, 1.0, 1.0)
    assert torch.equal(got.x, want.x) and torch.equal(got.kernel, want.kernel)
    assert (got.x[2] == 0).all()


def test_it_is_the_routers_transpose(lib):
    """Central differences of the float64 loss through the whole router (tokens, kernel and
    bias, the picks held), along random directions, against the op's gradients on what `route`
    itself returned. float32 sums in both; the kernel's and tokens' gradients are bfloat16, each
    element off by half a step at most, random in sign along a random direction: 6 standard
    deviations of their sum."""
    from bux_amd import router as r
    g = torch.Generator().manual_seed(11)
    t, d, n, scored, k = 96, 256, 36, 32, 4
    x = torch.randn(t, d, generator=g).to(BF16).cuda()
    kernel = (0.05 * torch.randn(d, n, generator=g)).to(BF16).cuda()
    bias = (0.1 * torch.randn(n, generator=g)).cuda()
    out = r.route(x, kernel, top_k=k, scored=scored, bias=bias, router_logit_scale=0.7,
                  routed_scaling_factor=2.5, with_logits=True)
    v = {"idx": out.idx, "logits": out.logits, "d_scores": None, "d_logits": None, "dz": None,
         "d_weights": torch.randn(t, k, generator=g).to(BF16).cuda(),
         "d_sinks": torch.randn(t, n - scored, generator=g).to(BF16).cuda()}
    got = r.route_backward(x, kernel, out.idx, out.logits, v["d_weights"], scored=scored,
                           router_logit_scale=0.7, routed_scaling_factor=2.5, d_sinks=v["d_sinks"])

    def loss(x, kernel, bias):
        return float(_loss((x @ kernel + bias) * 0.7, v, scored, "softmax", True, 2.5))

    at = {"x": x.double(), "kernel": kernel.double(), "bias": bias.double()}
    step = 1e-5
    for which, grad in (("x", got.x), ("kernel", got.kernel), ("bias", got.bias)):
        u = torch.randn(at[which].shape, generator=g, dtype=F64).cuda()
        up, down = dict(at), dict(at)
        up[which], down[which] = at[which] + step * u, at[which] - step * u
        want = (loss(**up) - loss(**down)) / (2 * step)
        terms = grad.double() * u
        rounding = 0 if which == "bias" else 6 * HALF_STEP * float(terms.square().sum().sqrt())
        # logits of float32 sums move G by some 2^-20; the differences are good to 1e-6
        assert abs(float(terms.sum()) - want) <= rounding + 1e-4 * float(terms.abs().sum()) / 10, which


def test_leading_dimensions_repeats_and_what_lies_past(lib):
    v = _inputs(300, 160, 40, 40, 4, seed=12, dz=True, scores=True)
    a = _run(v, 40, "softmax", True, 1.0, 1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    cube = {key: x if x is None or key == "kernel" else x.view(3, 100, x.shape[-1])
            for key, x in v.items()}
    with torch.cuda.stream(side):
        b = _run(cube, 40, "softmax", True, 1.0, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a.x.view(3, 100, 160), b.x)
    assert torch.equal(a.kernel, b.kernel) and torch.equal(a.bias, b.bias)
    # through the C ABI into buffers with more behind them
    t, d, n = 300, 160, 40
    dx = torch.full((t * d + 64,), 7.0, dtype=BF16, device="cuda")
    dk = torch.full((d * n + 64,), 7.0, dtype=BF16, device="cuda")
    db = torch.full((n + 8,), 7.0, device="cuda")
    need = lib.bux_route_backward_workspace_size(t, d, n)
    ws = torch.full((need + 256,), 9, dtype=torch.uint8, device="cuda")
    p = (lambda x: x.data_ptr())
    _lib.check(lib.bux_route_backward(
        p(v["x"]), p(v["kernel"]), t, d, n, 1.0, 0, 40, p(v["idx"]), 4, 1, 1.0, p(v["logits"]),
        p(v["d_weights"]), None, p(v["d_scores"]), None, p(v["dz"]), p(dx), p(dk), p(db), p(ws),
        need, None))
    assert torch.equal(dx[:t * d].view(t, d), a.x) and (dx[t * d:] == 7).all()
    assert torch.equal(dk[:d * n].view(d, n), a.kernel) and (dk[d * n:] == 7).all()
    assert torch.equal(db[:n], a.bias) and (db[n:] == 7).all()
    assert (ws[need:] == 9).all()


def test_in_a_graph(lib):
    v = _inputs(260, 272, 72, 64, 4, seed=13, dz=True, sinks=True)

    def step():
        return _run(v, 64, "softmax", True, 1.0, 2.5)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (20, 21, 22):
        for key, x in _inputs(260, 272, 72, 64, 4, seed=seed, dz=True, sinks=True).items():
            if x is not None:
                v[key].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(got.x, want.x) and torch.equal(got.kernel, want.kernel)
        assert torch.equal(got.bias, want.bias)


def test_tokens_at_any_element(lib):
    """Tokens and their gradient that begin at an odd element (a slice's): copied, not misread."""
    v = _inputs(40, 48, 24, 24, 3, seed=15, dz=True)
    want = _run(v, 24, "softmax", True, 1.0, 1.0)
    for key in ("x", "dz", "kernel"):
        buf = torch.zeros(v[key].numel() + 3, dtype=BF16, device="cuda")
        buf[3:].copy_(v[key].view(-1))
        v[key] = buf[3:].view(v[key].shape)
    got = _run(v, 24, "softmax", True, 1.0, 1.0)
    assert torch.equal(got.x, want.x) and torch.equal(got.kernel, want.kernel)


def test_a_workspace_of_nan(lib):
    """What the workspace holds on entry reaches no output (its padding rows among it)."""
    t, d, n = 37, 48, 20
    v = _inputs(t, d, n, n, 3, seed=16)
    want = _run(v, n, "softmax", True, 1.0, 1.0)
    need = lib.bux_route_backward_workspace_size(t, d, n)
    ws = torch.full((need // 2 + 1,), float("nan"), dtype=BF16, device="cuda")
    dx, dk = torch.empty_like(v["x"]), torch.empty_like(v["kernel"])
    p = (lambda x: x.data_ptr())
    _lib.check(lib.bux_route_backward(
        p(v["x"]), p(v["kernel"]), t, d, n, 1.0, 0, n, p(v["idx"]), 3, 1, 1.0, p(v["logits"]),
        p(v["d_weights"]), None, None, None, None, p(dx), p(dk), None, p(ws), need, None))
    assert torch.equal(dx, want.x) and torch.equal(dk, want.kernel)


def test_refusals(lib):
    from bux_amd import router as r
    v = _inputs(8, 32, 16, 14, 2, seed=14)

    def call(**kw):
        a = {**{key: v[key] for key in ("x", "kernel", "idx", "logits", "d_weights")}, "scored": 14, **kw}
        return r.route_backward(a.pop("x"), a.pop("kernel"), a.pop("idx"), a.pop("logits"),
                                a.pop("d_weights"), **a)

    call()
    with pytest.raises(TypeError, match="bfloat16"):
        call(x=v["x"].float())
    with pytest.raises(ValueError, match="idx"):
        call(idx=v["idx"].long())
    with pytest.raises(ValueError, match="logits"):
        call(logits=v["logits"][:, :15].contiguous())
    with pytest.raises(ValueError, match="d_weights"):
        call(d_weights=v["d_weights"].float())
    with pytest.raises(ValueError, match="d_sinks"):
        call(d_sinks=v["d_weights"].float())
    with pytest.raises(ValueError, match="scored"):
        call(scored=17)
    with pytest.raises(ValueError, match="router"):
        call(router="tanh")
    with pytest.raises(ValueError, match="kernel"):
        call(kernel=v["kernel"][:16].contiguous())
    with pytest.raises(ValueError, match="dz"):
        call(dz=v["x"][:4])
    with pytest.raises(ValueError, match="d=24"):
        call(x=v["x"][:, :24].contiguous(), kernel=v["kernel"][:24].contiguous())
