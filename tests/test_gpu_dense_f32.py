"""float32 dense products of enough columns for tiles of 128 x 128, where the small shapes of
test_gpu_dense.py take 128 x 64: every layout and epilogue, whole and with K in parts, odd edges.
Against the formulas in float64, on the GPU, within bounds counted beforehand (tests/_dense.py)."""

import pytest
import torch

from _dense import F32, F64, V, act, times, units
from _util import announce

pytestmark = pytest.mark.gpu

# m, k, n: the product whole, in 3 parts, in many; then its gradients to x and to w, whole
SHAPES = [(2701, 71, 2699), (1409, 261, 1409), (70, 2700, 2701), (2700, 2701, 69), (40, 3001, 2300)]


def _randn(g, *shape, scale=1.0):
    return scale * torch.randn(*shape, generator=g, device="cuda")


def _v(t):
    return V(t.to(F64))


@pytest.mark.parametrize("transposed", [False, True], ids=["", "transposed"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_product_and_its_gradients(lib, shape, transposed):
    from bux_amd import dense

    m, k, n = shape
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    x, w = _randn(g, m, k), _randn(g, *((n, k) if transposed else (k, n)), scale=k ** -0.5)
    b, r, dy = _randn(g, n), _randn(g, m, n), _randn(g, m, n, scale=0.1)
    wv = _v(w).t() if transposed else _v(w)
    z = _v(x) @ wv
    for bias, a, residual in ((None, None, None), (b, "swish", r)):
        announce("dense float32", shape, transposed, a)
        got = dense.product(x, w, bias, a, residual, transposed, with_product=a is not None)
        zb = z if bias is None else z + _v(bias)
        y = act(a, zb, F32)[0]
        y = y if residual is None else y + _v(residual)
        y.rounded(F32).holds(got.out, "out")
        if got.product is not None:
            zb.rounded(F32).holds(got.product, "product")
    announce("dense float32 backward", shape, transposed)
    got = dense.product_backward(dy, x, w, transposed=transposed)
    (_v(dy) @ wv.t()).rounded(F32).holds(got.x, "x")
    dw = _v(x).t() @ _v(dy)
    (dw.t() if transposed else dw).rounded(F32).holds(got.w, "w")


@pytest.mark.parametrize("gated", [True, False], ids=["gated", "plain"])
@pytest.mark.parametrize("shape", [(2701, 71, 2699), (1409, 261, 1409)], ids=str)
def test_block(lib, shape, gated):
    from bux_amd import mlp
    from bux_amd.moe import Ffn

    m, d, f = shape
    p = 2 if gated else 1
    g = torch.Generator(device="cuda").manual_seed(m + d + f)
    x, dy = _randn(g, m, d), _randn(g, m, d, scale=0.1)
    up, down = _randn(g, d, f, p, scale=d ** -0.5), _randn(g, f, d, scale=f ** -0.5)
    ub = _randn(g, f, p, scale=0.5)
    ffn = Ffn("swish", 2.0, 1.0)
    announce("mlp float32", shape, gated)
    r = mlp.feed_forward(x, up, down, ffn, ub)
    z = _v(x) @ V(up.to(F64).view(d, f * p)) + V(ub.to(F64).view(-1))
    z = V(z.v.view(m, f, p), z.e.view(m, f, p))
    z.rounded(F32).holds(r.saved.projected, "projected")
    units(ffn, z, gated, F32)[0].rounded(F32).holds(r.saved.h, "h")
    (_v(r.saved.h) @ _v(down)).rounded(F32).holds(r.out, "out")
    got = mlp.feed_forward_backward(dy, r.saved, up, down, ffn)
    dh = _v(dy) @ _v(down).t()
    _, du, dg = units(ffn, _v(r.saved.projected), gated, F32)
    parts = [times(dh, s) for s in (du, dg)[:p]]
    dp = V(torch.stack([q.v for q in parts], -1).view(m, f * p),
           torch.stack([q.e for q in parts], -1).view(m, f * p)).rounded(F32)
    (dp @ V(up.to(F64).view(d, f * p)).t()).rounded(F32).holds(got.x, "dx")
    dup = (_v(x).t() @ dp).rounded(F32)
    V(dup.v.view(d, f, p), dup.e.view(d, f, p)).holds(got.up, "dup")
    (_v(r.saved.h).t() @ _v(dy)).rounded(F32).holds(got.down, "ddown")
