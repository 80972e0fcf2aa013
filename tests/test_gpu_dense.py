"""Dense products with their epilogue (bux_amd.dense) and their backward against the formulas in
float64, within bounds counted beforehand (tests/_dense.py)."""

import pytest
import torch

from _dense import BF16, F32, F64, V, act, randn
from _util import announce

pytestmark = pytest.mark.gpu

# m, k, n: one of each, less than a load of 8, tiles' edges either way, odd rows, few rows with a
# long K (K in parts), no rows, whole tiles
SHAPES = [(1, 1, 1), (1, 7, 9), (3, 64, 8), (1, 2048, 256), (17, 300, 33), (33, 129, 130),
          (128, 64, 128), (129, 65, 257), (64, 4100, 72), (200, 1443, 1027), (300, 512, 264),
          (0, 64, 32), (256, 256, 512), (513, 96, 520), (16, 7168, 96), (5, 96, 2880),
          # few rows: one to four blocks of 16, K in parts and whole, cut steps, columns of no whole
          # 64s, enough columns for one part
          (16, 520, 264), (20, 1032, 264), (40, 2048, 1000), (48, 1000, 4104), (64, 4096, 136),
          (64, 72, 12296), (65, 512, 64)]


def _make(g, dtype, m, k, n, transposed=False):
    x = randn(g, m, k).to(dtype).cuda()
    w = (randn(g, *((n, k) if transposed else (k, n))) / max(k, 1) ** 0.5).to(dtype).cuda()
    return x, w, (0.5 * randn(g, n)).to(dtype).cuda(), randn(g, m, n).to(dtype).cuda()


def _v(t):
    return None if t is None else V(t.cpu().to(F64))


def _forward(x, w, b, a, r, transposed):
    wv = _v(w).t() if transposed else _v(w)
    z = _v(x) @ wv + _v(b)
    return z, act(a, z, x.dtype)[0] + _v(r)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("transposed", [False, True], ids=["", "transposed"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_product(lib, shape, transposed, dtype):
    from bux_amd import dense

    m, k, n = shape
    g = torch.Generator().manual_seed(m + 7 * k + 31 * n)
    x, w, b, r = _make(g, dtype, m, k, n, transposed)
    for bias, a, residual in ((None, None, None), (b, "swish", r), (None, "gelu_tanh", None),
                              (b, None, r), (None, "relu2", r)):
        announce("dense product", shape, dtype, transposed, a)
        got = dense.product(x, w, bias, a, residual, transposed, with_product=True)
        z, y = _forward(x, w, bias, a, residual, transposed)
        z.rounded(dtype).holds(got.product, "product")
        y.rounded(dtype).holds(got.out, "out")
        bare = dense.product(x, w, bias, a, residual, transposed)
        assert bare.product is None and torch.equal(bare.out, got.out)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("kind", ["swish", "quick_gelu", "relu", "relu2", "gelu", "gelu_tanh",
                                  "sigmoid", "tanh", "softplus", "situ"])
def test_every_activation(lib, kind, dtype):
    from bux_amd import dense

    g = torch.Generator().manual_seed(3)
    for m, k, n in ((37, 65, 131), (256, 64, 512)):
        x, w, b, r = _make(g, dtype, m, k, n)
        x = x * 3
        announce("dense activation", kind, dtype, m)
        got = dense.product(x, w, b, kind, r, with_product=True)
        _, y = _forward(x, w, b, kind, r, False)
        y.rounded(dtype).holds(got.out, "out")
        dy = (0.1 * randn(g, m, n)).to(dtype).cuda()
        grads = dense.product_backward(dy, x, w, kind, got.product, bias=True)
        _, s = act(kind, _v(got.product), dtype)
        dz = V(_v(dy).v * s.v, _v(dy).v.abs() * s.e + 4 * 2.0 ** -24 * (_v(dy).v * s.v).abs())
        dz.sum0().rounded(dtype).holds(grads.bias, "bias")
        kept = dz.rounded(dtype)  # dz between the kernels
        (kept @ _v(w).t()).rounded(dtype).holds(grads.x, "x")
        (_v(x).t() @ kept).rounded(dtype).holds(grads.w, "w")


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("transposed", [False, True], ids=["", "transposed"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_backward(lib, shape, transposed, dtype):
    from bux_amd import dense

    m, k, n = shape
    g = torch.Generator().manual_seed(2 * m + 7 * k + 31 * n)
    x, w, _, dy = _make(g, dtype, m, k, n, transposed)
    announce("dense backward", shape, dtype, transposed)
    got = dense.product_backward(dy, x, w, transposed=transposed, bias=True)
    wv = _v(w) if transposed else _v(w).t()
    (_v(dy) @ wv).rounded(dtype).holds(got.x, "x")
    dw = _v(x).t() @ _v(dy)
    (dw.t() if transposed else dw).rounded(dtype).holds(got.w, "w")
    _v(dy).sum0().rounded(dtype).holds(got.bias, "bias")
    assert dense.product_backward(dy, x, w, transposed=transposed).bias is None


def test_gradients_against_differences(lib):
    """The float32 gradients along a random direction, against a central difference of the
    formula in float64: its step of 1e-4 leaves a third derivative's 1e-8 of the loss's scale."""
    from bux_amd import dense

    g = torch.Generator().manual_seed(11)
    m, k, n = 37, 45, 51
    x, w, b, r = _make(g, F32, m, k, n)
    dy = randn(g, m, n).to(F32).cuda()
    got = dense.product(x, w, b, "gelu", r, with_product=True)
    grads = dense.product_backward(dy, x, w, "gelu", got.product, bias=True)
    v = [randn(g, m, k), randn(g, k, n), randn(g, n)]

    def loss(e):
        z = (x.cpu().to(F64) + e * v[0]) @ (w.cpu().to(F64) + e * v[1]) + b.cpu().to(F64) + e * v[2]
        return (dy.cpu().to(F64) * (z * torch.special.ndtr(z))).sum()

    want = (loss(1e-4) - loss(-1e-4)) / 2e-4
    parts = [(gr.cpu().to(F64) * d) for gr, d in zip((grads.x, grads.w, grads.bias), v)]
    scale = sum(p.abs().sum() for p in parts)
    # float32 gradients: under 100 roundings each, relative to the terms' magnitudes
    assert abs(sum(p.sum() for p in parts) - want) <= (200 * 2.0 ** -24 + 1e-7) * scale


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_operands_at_an_odd_element(lib, dtype):
    """Contiguous tensors that begin one element past any alignment, between values that are no
    numbers, which no result may hold."""
    from bux_amd import dense

    g = torch.Generator().manual_seed(5)

    def odd(t):
        flat = torch.full((t.numel() + 18,), float("nan"), dtype=dtype, device="cuda")
        flat[9:9 + t.numel()] = t.reshape(-1)
        return flat[9:9 + t.numel()].view(t.shape)

    for m, k, n in ((256, 128, 512), (70, 96, 72), (2, 4096, 64)):
        x, w, b, r = (odd(t) for t in _make(g, dtype, m, k, n))
        assert x.data_ptr() % 4 == 2 or dtype == F32
        announce("dense odd element", m, k, n, dtype)
        got = dense.product(x, w, b, "swish", r)
        _forward(x, w, b, "swish", r, False)[1].rounded(dtype).holds(got.out, "out")
        dy = odd(r.clone())
        grads = dense.product_backward(dy, x, w, bias=True)
        (_v(dy) @ _v(w).t()).rounded(dtype).holds(grads.x, "x")
        (_v(x).t() @ _v(dy)).rounded(dtype).holds(grads.w, "w")


def test_a_number_that_is_none_stays_in_its_row_and_column(lib):
    from bux_amd import dense

    g = torch.Generator().manual_seed(6)
    for m, k, n in ((200, 100, 150), (300, 256, 512), (4, 2048, 96)):
        x, w, _, _ = _make(g, BF16, m, k, n)
        clean = dense.product(x, w).out
        x[1, k - 1], w[k - 1, 2] = float("nan"), float("inf")
        got = dense.product(x, w).out
        rows = torch.arange(m, device="cuda") != 1
        cols = torch.arange(n, device="cuda") != 2
        assert torch.equal(got[rows][:, cols], clean[rows][:, cols])
        assert got[1].isnan().all() and (~got[:, 2].isfinite()).all()


def test_rows_of_any_leading_dimensions_and_no_rows(lib):
    from bux_amd import dense

    g = torch.Generator().manual_seed(7)
    x, w, b, r = _make(g, BF16, 24, 96, 80)
    flat = dense.product(x, w, b, "swish", r)
    deep = dense.product(x.view(2, 3, 4, 96), w, b, "swish", r.view(2, 3, 4, 80))
    assert deep.out.shape == (2, 3, 4, 80) and torch.equal(deep.out.view(24, 80), flat.out)
    one = dense.product(x[5], w, b, "swish", r[5])
    assert one.out.shape == (80,)
    none = dense.product_backward(x.new_zeros(0, 80), x.new_zeros(0, 96), w, bias=True)
    assert none.x.shape == (0, 96) and not none.w.any() and not none.bias.any()


def test_another_stream(lib):
    from bux_amd import dense

    g = torch.Generator().manual_seed(8)
    x, w, b, r = _make(g, BF16, 64, 4100, 72)
    want = dense.product(x, w, b, "swish", r).out
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = dense.product(x, w, b, "swish", r).out
    s.synchronize()
    assert torch.equal(got, want)


def test_refusals(lib):
    from bux_amd import dense

    x = torch.zeros(4, 32, dtype=BF16, device="cuda")
    w = torch.zeros(32, 16, dtype=BF16, device="cuda")
    with pytest.raises(TypeError, match="float16"):
        dense.product(x.half(), w.half())
    with pytest.raises(TypeError, match="float32"):
        dense.product(x, w.float())
    with pytest.raises(ValueError, match="rows of 32"):
        dense.product(x[:, :16].contiguous(), w)
    with pytest.raises(ValueError, match="rows of 16"):
        dense.product(x, w, transposed=True)
    with pytest.raises(ValueError, match="bias"):
        dense.product(x, w, bias=x[0])
    with pytest.raises(ValueError, match="residual"):
        dense.product(x, w, residual=x)
    with pytest.raises(ValueError, match="no activation"):
        dense.product(x, w, activation="softmax")
    with pytest.raises(ValueError, match="contiguous"):
        dense.product(x, w.t().contiguous().t())
    with pytest.raises(ValueError, match="on cpu"):
        dense.product(x, w.cpu())
    with pytest.raises(ValueError, match="kernel"):
        dense.product(x, w[None])
    with pytest.raises(ValueError, match="kept product"):
        dense.product_backward(x[:, :16].contiguous(), x, w, "swish")
    with pytest.raises(ValueError, match="dy"):
        dense.product_backward(x, x, w)
    with pytest.raises(ValueError, match="rows"):
        dense.weight_grad(x, x[:2])
