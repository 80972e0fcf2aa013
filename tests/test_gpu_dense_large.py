"""Dense products of enough 256 x 256 tiles to run on the large tiles' kernel: every layout and
epilogue, K of one unit to many, whole and cut, tiles cut by the rows' and columns' ends, several
tiles a workgroup. Against the formulas in float64, on the GPU, within bounds counted beforehand
(tests/_dense.py)."""

import pytest
import torch

from _dense import BF16, F64, V, act, kept, times, units
from _util import announce

pytestmark = pytest.mark.gpu

# m, k, n
SHAPES = [(4352, 8, 4608), (4100, 64, 4104), (3400, 72, 4104), (4352, 128, 4608), (4096, 192, 4096),
          (4097, 200, 3928), (5000, 320, 2824), (260, 456, 51208), (33000, 136, 520),
          # K in parts, whole and cut
          (1024, 4096, 4096), (1000, 4104, 4000), (520, 7168, 4096)]


def _randn(g, *shape, scale=1.0):
    return (scale * torch.randn(*shape, generator=g, device="cuda")).to(BF16)


def _v(t):
    return V(t.to(F64))


@pytest.mark.parametrize("transposed", [False, True], ids=["", "transposed"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_product(lib, shape, transposed):
    from bux_amd import dense

    m, k, n = shape
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    x, w = _randn(g, m, k), _randn(g, *((n, k) if transposed else (k, n)), scale=k ** -0.5)
    b, r = _randn(g, n), _randn(g, m, n)
    z = _v(x) @ (_v(w).t() if transposed else _v(w))
    for bias, a, residual in ((None, None, None), (b, "swish", r)):
        announce("dense large", shape, transposed, a)
        got = dense.product(x, w, bias, a, residual, transposed, with_product=a is not None)
        zb = z if bias is None else z + _v(bias)
        y = act(a, zb, BF16)[0]
        y = y if residual is None else y + _v(residual)
        y.rounded(BF16).holds(got.out, "out")
        if got.product is not None:
            zb.rounded(BF16).holds(got.product, "product")


@pytest.mark.parametrize("shape", [(8, 4352, 4608), (72, 4104, 3400), (200, 3928, 4104),
                                   (456, 260, 51208), (1001, 4096, 4096), (4096, 1024, 4096),
                                   (8200, 2048, 1032)], ids=str)
def test_weight_grad(lib, shape):
    from bux_amd import dense

    m, k, n = shape
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    x, dy = _randn(g, m, k), _randn(g, m, n, scale=0.1)
    announce("dense large wgrad", shape)
    (_v(x).t() @ _v(dy)).rounded(BF16).holds(dense.weight_grad(x, dy), "dw")


@pytest.mark.parametrize("gated", [True, False], ids=["gated", "plain"])
@pytest.mark.parametrize("shape", [(4100, 136, 4104), (8200, 64, 1928), (3000, 264, 5000),
                                   (1024, 4096, 2048)], ids=str)
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
    announce("mlp large", shape, gated)
    r = mlp.feed_forward(x, up, down, ffn, ub)
    z = _v(x) @ V(up.to(F64).view(d, f * p)) + V(ub.to(F64).view(-1))
    z = V(z.v.view(m, f, p), z.e.view(m, f, p))
    z.rounded(BF16).holds(r.saved.projected, "projected")
    V(z.v, z.e + 2.0 ** -15 * (z.v.abs() + z.e)).holds(kept(r.saved), "24 bits")
    units(ffn, z, gated, BF16)[0].rounded(BF16).holds(r.saved.h, "h")
    (_v(r.saved.h) @ _v(down)).rounded(BF16).holds(r.out, "out")
    got = mlp.feed_forward_backward(dy, r.saved, up, down, ffn)
    dh = _v(dy) @ _v(down).t()
    _, du, dg = units(ffn, _v(kept(r.saved)), gated, BF16)
    parts = [times(dh, s) for s in (du, dg)[:p]]
    dp = V(torch.stack([q.v for q in parts], -1).view(m, f * p),
           torch.stack([q.e for q in parts], -1).view(m, f * p)).rounded(BF16)
    (dp @ V(up.to(F64).view(d, f * p)).t()).rounded(BF16).holds(got.x, "dx")
    dup = (_v(x).t() @ dp).rounded(BF16)
    V(dup.v.view(d, f, p), dup.e.view(d, f, p)).holds(got.up, "dup")
    (_v(r.saved.h).t() @ _v(dy)).rounded(BF16).holds(got.down, "ddown")


def test_nan_stays_in_its_row(lib):
    from bux_amd import dense

    g = torch.Generator(device="cuda").manual_seed(1)
    m, k, n = 4100, 72, 4104
    x, w = _randn(g, m, k), _randn(g, k, n)
    clean = dense.product(x, w).out
    x[1], x[4099] = float("nan"), float("inf")
    got = dense.product(x, w).out
    rows = torch.ones(m, dtype=torch.bool, device="cuda")
    rows[1] = rows[4099] = False
    assert torch.equal(got[rows], clean[rows]) and got[1].isnan().all()
    assert (~got[4099].isfinite()).all()
