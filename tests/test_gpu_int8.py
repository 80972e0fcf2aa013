"""The experts' products in 8-bit integers (bux_amd.grouped_int8, moe.experts_int8).

Everything but the activation has an exact answer: codes by the quotient in float64 (127 x is
exact there; a quotient that is no tie lies 2^-33 of it from one at least, over float64's
rounding), scales and products by float32 operations in the same order, sums as integers. So
these compare bit for bit. The products of real values lie within what the rounding of the
codes allows, half a code of either operand.
"""

import ctypes

import numpy as np
import pytest
import torch

from _util import announce
from bux_amd import _lib

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _codes(x: torch.Tensor) -> tuple[np.ndarray, np.ndarray]:
    """Codes (r, c) and scales (r,) of finite rows, on the host."""
    v = x.detach().double().cpu().numpy()
    top = np.abs(v).max(-1, keepdims=True) if v.shape[-1] else np.zeros((v.shape[0], 1))
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.rint(np.where(top > 0, 127.0 * v / top, 0.0))
    return q.astype(np.int8), (top[:, 0].astype(np.float32) / np.float32(127))


def _untiled(t, cols):
    """An `Int8`'s codes row-major (..., r, cols) and scales on the host, its padding checked."""
    v = t.values.cpu().numpy()
    n = v.ndim - 3
    v = np.swapaxes(v, n, n + 1)
    v = v.reshape(*v.shape[:n + 1], -1)
    assert (v[..., cols:] == 0).all(), "codes past the columns are not 0"
    return v[..., :cols], t.scales.cpu().numpy()


def _normal(seed, *shape, dtype=BF16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (130, 100), (9, 1000), (4, 1024),
                                       (7, 2048), (6, 2050), (5, 4096), (3, 7168), (2, 8192),
                                       (2, 8200), (2, 9001), (0, 64)])
def test_rows(lib, rows, cols, dtype):
    from bux_amd import grouped_int8 as g8
    announce("int8 rows", rows, cols, dtype)
    x = _normal(rows + cols, rows, cols, dtype=dtype)
    if rows > 1:
        x[1] = 0  # a row of zeros
    if rows > 2:
        x[2] *= 1e-3
        x[2, cols // 2] = -50.0  # one value far above the rest
    height = rows + 5
    q = g8.quantized(x, height=height)
    codes, scales = _untiled(q, cols)
    want, ws = _codes(x)
    assert q.values.shape == (-(-cols // 128) * 2, height, 64)
    assert np.array_equal(codes[:rows], want) and np.array_equal(scales[:rows], ws)
    assert (codes[rows:] == 0).all() and (scales[rows:] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("cols", [*range(8, 17), *range(249, 259), *range(505, 515), 1017, 4099])
def test_rows_of_every_last_part(lib, cols, dtype):
    """Rows whose last 8 columns are cut short anywhere, at any element of a buffer with NaN on
    either side; the largest value in the row's first or last column."""
    from bux_amd import grouped_int8 as g8
    announce("int8 last part", cols, dtype)
    rows = 21
    for shift in (0, 1, 3, 8):
        buffer = torch.full((rows * cols + 16,), float("nan"), dtype=dtype, device="cuda")
        x = buffer[shift:shift + rows * cols].view(rows, cols)
        x.copy_(_normal(cols, rows, cols, dtype=dtype))
        x[::2, -1], x[1::2, 0] = 9.0, -9.0
        codes, scales = _untiled(g8.quantized(x), cols)
        want, ws = _codes(x)
        assert np.array_equal(codes, want) and np.array_equal(scales, ws)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_every_bfloat16_under_many_scales(lib, dtype):
    """Rows of every finite bfloat16 up to the row's largest, over largest values of all kinds of
    mantissas and from the smallest subnormal to the largest: ties and near ties among them."""
    from bux_amd import grouped_int8 as g8
    bits = np.arange(0, 0x7F80, dtype=np.uint16)
    tops = sorted({0x0001, 0x0003, 0x007F, 0x0080, 0x00FE, 0x1FFF, 0x7F7F, 0x7F00, 0x3F80, 0x3F81,
                   0x3FAA, 0x3FFF, 0x42FE, 0x42FF, 0x437F, 0x0D80, 0x0D7F,
                   *np.random.default_rng(0).integers(1, 0x7F80, 24).tolist()})
    x = np.zeros((len(tops), 2 * len(bits)), np.uint16)
    for r, top in enumerate(tops):
        row = np.where(bits <= top, bits, 0)
        x[r] = np.concatenate([row, row | 0x8000])
    x = torch.from_numpy(x.view(np.int16)).view(BF16).to(dtype)
    codes, scales = _untiled(g8.quantized(x.cuda()), x.shape[1])
    want, ws = _codes(x)
    assert np.array_equal(codes, want)
    assert np.array_equal(scales, ws)


def test_float32_ties_and_their_neighbours(lib):
    """Values at (n + 1/2) m / 127 for a largest value m of 127 2^j (ties exactly) and the
    float32 on either side of each; and values around the ties of odd largest values."""
    from bux_amd import grouped_int8 as g8
    rows = []
    for m in (127.0, 127.0 / 8, 127.0 * 2**20, 1.0, 3.3333, 0.7, 1e-30, 3e38, 1e-40):
        m = np.float32(m)
        ties = ((np.arange(0, 127) + 0.5) * np.float64(m) / 127).astype(np.float32)
        row = np.concatenate([ties, np.nextafter(ties, np.float32(0)),
                              np.nextafter(ties, np.float32(np.inf))])
        rows.append(np.concatenate([[m], np.minimum(row, m), -np.minimum(row, m)]))
    x = torch.from_numpy(np.stack(rows).astype(np.float32))
    codes, scales = _untiled(g8.quantized(x.cuda()), x.shape[1])
    want, ws = _codes(x)
    assert np.array_equal(codes, want) and np.array_equal(scales, ws)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("cols", [96, 300, 8200, 61])
def test_infinities_and_nan(lib, cols, dtype):
    from bux_amd import grouped_int8 as g8
    x = _normal(1, 4, cols, dtype=dtype)
    x[0, cols - 1], x[1, 0], x[2, 3] = float("nan"), float("inf"), -float("inf")
    x[2, 4] = float("nan")
    codes, scales = _untiled(g8.quantized(x), cols)
    assert np.isnan(scales[0]) and np.isposinf(scales[1]) and np.isnan(scales[2])
    assert (codes[:3] == 0).all()
    want, ws = _codes(x[3:])
    assert np.array_equal(codes[3:], want) and scales[3] == ws[0]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_rows_by_index(lib, dtype):
    """Picks' tokens, some outside them; from `filled` on, and past the picks, zeros."""
    from bux_amd import grouped_int8 as g8
    x = _normal(2, 10, 200, dtype=dtype)
    index = torch.tensor([0, 39, 7, -1, 40, 2**31 - 1, -2**31, 13, 13, 22], dtype=torch.int32).cuda()
    want, ws = _codes(x)
    for filled in (None, 9, 0, 20, -3):
        f = None if filled is None else torch.tensor([filled], dtype=torch.int32).cuda()
        codes, scales = _untiled(g8.quantized(x, f, index, 4, 16), 200)
        for i in range(16):
            pick = int(index[i]) if i < (10 if filled is None else max(0, min(filled, 10))) else -1
            token = pick // 4 if pick >= 0 else 99
            if token < 10:
                assert np.array_equal(codes[i], want[token]) and scales[i] == ws[token]
            else:
                assert (codes[i] == 0).all() and scales[i] == 0


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("cols", [1003, 3968])
def test_many_rows_by_index(lib, cols, dtype):
    """Enough rows of few enough tokens that each token is quantized once: the same codes, for
    any index (repeated, unordered, outside the tokens), any `filled`."""
    from bux_amd import grouped_int8 as g8
    tokens, div = 900, 3
    rows = -(-2**25 // cols) + 77
    announce("int8 many rows", cols, dtype)
    assert lib.bux_int8_quantize_workspace_size(tokens, rows, cols) > 0
    x = _normal(8, tokens, cols, dtype=dtype)
    x[5], x[6, 1] = 0, float("nan")
    g = torch.Generator().manual_seed(9)
    index = torch.randint(-40, tokens * div + 40, (rows,), generator=g, dtype=torch.int32)
    index[:4] = torch.tensor([2**31 - 1, -2**31, tokens * div - 1, tokens * div])
    index = index.cuda()
    filled = torch.tensor([rows - 1000], dtype=torch.int32).cuda()
    got = g8.quantized(x, filled, index, div, rows + 300)
    one = g8.quantized(x)
    token = torch.div(index, div, rounding_mode="floor").long()
    live = (index >= 0) & (token < tokens) & (torch.arange(rows, device="cuda") < rows - 1000)
    token = torch.where(live, token, 0)
    values = torch.where(live[None, :, None], one.values[:, token], 0)
    assert torch.equal(got.values[:, :rows], values) and (got.values[:, rows:] == 0).all()
    scales = torch.where(live, one.scales[token], 0.0)
    assert torch.equal(got.scales[:rows].view(torch.int32), scales.view(torch.int32))
    assert (got.scales[rows:] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("g,k,n", [(1, 1, 1), (2, 64, 64), (3, 100, 70), (2, 300, 129), (1, 1000, 4)])
def test_kernels_columns(lib, g, k, n, dtype):
    from bux_amd import grouped_int8 as g8
    announce("int8 columns", g, k, n, dtype)
    w = _normal(g + k + n, g, k, n, dtype=dtype)
    w[0, :, 0] = 0
    if n > 2:
        w[g - 1, 0, 2] = float("inf")
    codes, scales = _untiled(g8.quantized_kernels(w), k)
    assert codes.shape == (g, n, k) and scales.shape == (g, n)
    for i in range(g):
        t = w[i].t().contiguous()
        if n > 2 and i == g - 1:
            assert np.isposinf(scales[i, 2]) and (codes[i, 2] == 0).all()
            t[2] = 0
            codes[i, 2], scales[i, 2] = 0, 0
        want, ws = _codes(t)
        assert np.array_equal(codes[i], want) and np.array_equal(scales[i], ws)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("activation,gated", [("swish", True), ("quick_gelu", True), ("relu2", False),
                                              ("gelu", False), ("situ", True)])
@pytest.mark.parametrize("f", [4, 100, 768, 1028, 2880, 4100])
def test_the_activation_in_one_pass(lib, f, activation, gated, dtype):
    """weighted_units, then quantized: the same bits."""
    from bux_amd import grouped_int8 as g8, moe
    announce("int8 activation", f, activation, gated, dtype)
    m = 9
    ffn = moe.Ffn(activation, 7.0 if gated else None, 1.0 if gated else 0.0)
    projected = _normal(f, m, f, 2 if gated else 1, dtype=dtype, scale=3.0)
    weights = _normal(f + 1, m, dtype=dtype)
    weights[3] = 0
    filled = torch.tensor([7], dtype=torch.int32).cuda()
    got = moe.weighted_units_int8(ffn, projected, weights, filled, m + 4)
    want = g8.quantized(moe.weighted_units(ffn, projected, weights, filled), filled, height=m + 4)
    assert torch.equal(got.values, want.values) and torch.equal(got.scales, want.scales)


def _random_int8(seed, *lead, rows, k):
    """An Int8 of codes over the whole range, its padding 0, and codes row-major."""
    from bux_amd import grouped_int8 as g8
    g = torch.Generator().manual_seed(seed)
    chunks = -(-k // 128) * 2
    codes = torch.randint(-127, 128, (*lead, rows, k), generator=g, dtype=torch.int8)
    padded = torch.zeros(*lead, rows, chunks * 64, dtype=torch.int8)
    padded[..., :k] = codes
    tiled = padded.view(*lead, rows, chunks, 64).transpose(-3, -2).contiguous()
    scales = torch.rand(*lead, rows, generator=g) * 0.01 + 1e-4
    return g8.Int8(tiled.cuda(), scales.cuda()), codes


def _product(a, a_scales, b, b_scales, sizes, height, dtype, bias=None):
    """The products as the op's float32 operations give them, on the host."""
    groups, n, _ = b.shape
    y = torch.zeros(height, n, dtype=F32)
    row = 0
    for g, size in enumerate(sizes):
        size = min(max(size, 0), max(a.shape[0], height) - row)
        rows = min(size, height - row, a.shape[0] - row)
        if rows > 0:
            s = a[row:row + rows].double() @ b[g].double().t()  # exact: below 2^31
            v = s.float() * (a_scales[row:row + rows, None] * b_scales[g])
            y[row:row + rows] = v if bias is None else v + bias[g].float()
        row += size
    return y.to(dtype)


# groups, sizes (in sequence), rows of a past them, k, n
PRODUCTS = [
    ([1], 0, 1, 4),
    ([5, 0, 3], 2, 64, 12),
    ([1, 1, 1, 1, 1], 0, 130, 64),
    ([256], 0, 128, 256),
    ([257, 255, 1], 7, 200, 260),
    ([128, 129, 130], 0, 384, 516),
    ([0, 0, 600], 40, 700, 132),
    ([33, 64, 65, 31, 96], 3, 2048, 300),
    ([300, 20, 0, 500, 7], 100, 1000, 1024),
    ([0, 0], 9, 128, 8),
]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("biased", [False, True], ids=["", "biased"])
@pytest.mark.parametrize("case", PRODUCTS, ids=lambda c: f"{len(c[0])}x{sum(c[0])}x{c[2]}x{c[3]}")
def test_products(lib, case, biased, dtype):
    from bux_amd import grouped_int8 as g8
    sizes, past, k, n = case
    announce("int8 products", case, biased, dtype)
    m = sum(sizes) + past
    a, ac = _random_int8(k, rows=m, k=k)
    b, bc = _random_int8(n, len(sizes), rows=n, k=k)
    bias = _normal(3, len(sizes), n, dtype=dtype) if biased else None
    sz = torch.tensor(sizes, dtype=torch.int32).cuda()
    for height in sorted({m, m + 3, max(0, m - 5)}):
        y = g8.rows(a, b, sz, dtype, height, bias=bias)
        want = _product(ac, a.scales.cpu(), bc, b.scales.cpu(), sizes, height, dtype,
                        None if bias is None else bias.cpu())
        assert torch.equal(y.cpu(), want), (height, (y.cpu() != want).nonzero()[:5])


# few rows a group, some groups with many: sizes, rows of a past them, k, n
FEW = [
    ([1, 0, 2, 0, 1, 1], 0, 2048, 132),
    ([0] * 12 + [200] + [0] * 12, 3, 300, 68),
    ([300] + [1] * 30, 0, 96, 64),
    ([16, 17, 15, 31, 1, 0, 32, 33, 2, 0, 0, 0], 5, 1000, 260),
    ([0] * 5, 7, 128, 4),
]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("biased", [False, True], ids=["", "biased"])
@pytest.mark.parametrize("case", FEW, ids=lambda c: f"{len(c[0])}x{sum(c[0])}x{c[2]}x{c[3]}")
def test_products_of_few_rows_a_group(lib, case, biased, dtype):
    from bux_amd import grouped_int8 as g8
    sizes, past, k, n = case
    m = sum(sizes) + past
    announce("int8 products of few rows", case, biased, dtype)
    a, ac = _random_int8(k, rows=m, k=k)
    b, bc = _random_int8(n, len(sizes), rows=n, k=k)
    bias = _normal(3, len(sizes), n, dtype=dtype) if biased else None
    a.scales[sum(sizes):] = float("nan")  # past the groups
    if sizes[0] > 1:
        a.scales[1], ac[1] = float("inf"), 0
        a.values[:, 1] = 0
    sz = torch.tensor(sizes, dtype=torch.int32).cuda()
    buf = torch.full((m * n + 512 * n,), 7.0, dtype=dtype, device="cuda")
    for height in (m, m + 40):
        y = g8.rows(a, b, sz, dtype, height, bias=bias)
        want = _product(ac, a.scales.cpu(), bc, b.scales.cpu(), sizes, height, dtype,
                        None if bias is None else bias.cpu())
        if sizes[0] > 1:
            assert torch.isnan(y[1]).all()
            y[1], want[1] = 0, 0
        assert torch.equal(y.cpu(), want), (height, (y.cpu() != want).nonzero()[:5])
    from bux_amd import grouped_mxfp8
    tiles = grouped_mxfp8.tiles_of(sz, m, m)
    _lib.check(lib.bux_int8_grouped_rows_listed(
        a.values.data_ptr(), a.scales.data_ptr(), b.values.data_ptr(), b.scales.data_ptr(),
        tiles.buffer.data_ptr(), tiles.buffer.numel(), len(sizes), m, n, -(-k // 128) * 128, m,
        0 if dtype == BF16 else 1, None if bias is None else bias.data_ptr(),
        buf[256 * n:].data_ptr(), None))
    assert (buf[:256 * n] == 7).all() and (buf[256 * n + m * n:] == 7).all()


def test_both_kernels_give_the_same_bits(lib):
    """One product by either kernel: its rows in two groups, and those groups beside many empty
    ones (which kernel a call takes goes by its rows a group)."""
    from bux_amd import grouped_int8 as g8
    direct = lib.bux_int8_direct
    direct.argtypes, direct.restype = [ctypes.c_int64, ctypes.c_int32], ctypes.c_int
    m, n, k = 150, 196, 700
    assert not direct(m, 2) and direct(m, 40)
    assert [direct(160, 10), direct(161, 10)] == [1, 0]
    a, _ = _random_int8(1, rows=m, k=k)
    b, _ = _random_int8(2, 40, rows=n, k=k)
    two = g8.Int8(b.values[:2].contiguous(), b.scales[:2].contiguous())
    sizes = torch.zeros(40, dtype=torch.int32).cuda()
    sizes[:2] = torch.tensor([100, 50])
    for dtype in (BF16, F32):
        assert torch.equal(g8.rows(a, b, sizes, dtype), g8.rows(a, two, sizes[:2].contiguous(), dtype))


def test_the_largest_sums(lib):
    """K of 131072 codes of +-127: sums of 127^2 K, 2^31 less a 64th."""
    from bux_amd import grouped_int8 as g8
    k = 131072
    a = g8.Int8(torch.full((k // 64, 3, 64), 127, dtype=torch.int8, device="cuda"),
                torch.ones(3, device="cuda"))
    b = g8.Int8(torch.full((2, k // 64, 4, 64), 127, dtype=torch.int8, device="cuda"),
                torch.ones(2, 4, device="cuda"))
    b.values[1] = -127
    y = g8.rows(a, b, torch.tensor([2, 1], dtype=torch.int32).cuda(), F32)
    want = float(np.float32(127 * 127 * k))
    assert (y[:2] == want).all() and (y[2] == -want).all()


def test_bad_sizes_and_rows_behind(lib):
    """A negative size counts as 0, sizes past the rows stop there, and nothing is written
    outside y."""
    from bux_amd import grouped_int8 as g8, grouped_mxfp8
    k, n, m = 256, 68, 300
    a, ac = _random_int8(1, rows=m, k=k)
    b, bc = _random_int8(2, 4, rows=n, k=k)
    for sizes in ([100, -50, 60, 90], [200, 2**31 - 1, 5, 5], [2**31 - 1] * 4):
        sz = torch.tensor(sizes, dtype=torch.int32).cuda()
        tiles = grouped_mxfp8.tiles_of(sz, m, m)
        buf = torch.full((m * n + 2 * 256 * n,), 7.0, dtype=BF16, device="cuda")
        y = buf[256 * n:256 * n + m * n]
        _lib.check(lib.bux_int8_grouped_rows_listed(
            a.values.data_ptr(), a.scales.data_ptr(), b.values.data_ptr(), b.scales.data_ptr(),
            tiles.buffer.data_ptr(), tiles.buffer.numel(), 4, m, n, k, m, 0, None, y.data_ptr(), None))
        want = _product(ac, a.scales.cpu(), bc, b.scales.cpu(), sizes, m, BF16)
        assert torch.equal(y.view(m, n).cpu(), want)
        assert (buf[:256 * n] == 7).all() and (buf[256 * n + m * n:] == 7).all()


def test_a_row_that_is_not_a_number_stays_its_own(lib):
    from bux_amd import grouped_int8 as g8
    a, ac = _random_int8(1, rows=70, k=200)
    b, bc = _random_int8(2, 2, rows=72, k=200)
    sz = torch.tensor([40, 25], dtype=torch.int32).cuda()
    want = g8.rows(a, b, sz)
    a.scales[3], a.values[:, 3] = float("nan"), 0
    a.scales[50], a.values[:, 50] = float("inf"), 0
    a.scales[66:] = float("nan")  # past the groups
    y = g8.rows(a, b, sz)
    keep = [i for i in range(70) if i not in (3, 50)]
    assert torch.equal(y[keep], want[keep])
    assert torch.isnan(y[3]).all() and torch.isnan(y[50]).all() and (y[65:] == 0).all()


def test_a_list_of_other_dimensions_is_refused(lib):
    from bux_amd import grouped_int8 as g8, grouped_mxfp8
    a, _ = _random_int8(1, rows=64, k=128)
    b, _ = _random_int8(2, 2, rows=64, k=128)
    sz = torch.tensor([30, 20], dtype=torch.int32).cuda()
    with pytest.raises(ValueError, match="tile list"):
        g8.rows(a, b, sz, tiles=grouped_mxfp8.tiles_of(sz, 128, 64))
    tiles = grouped_mxfp8.tiles_of(sz, 128, 64)
    y = g8.rows(a, b, sz, tiles=grouped_mxfp8.TileList(tiles.buffer, 2, 64, 64))
    torch.cuda.synchronize()
    assert tiles.buffer.view(torch.int32)[4] == _lib.LIST_REFUSED and y.shape == (64, 64)


def test_products_of_real_values_lie_within_the_codes(lib):
    """|y - x w| <= sum over k of s_w/2 |x| + s_x/2 |w| + s_x s_w / 4 (half a code of each), and
    the float32 roundings of the scales and the product, 6 u of the magnitudes."""
    from bux_amd import grouped_int8 as g8
    x, w = _normal(5, 90, 500, dtype=F32), _normal(6, 2, 500, 64, dtype=F32)
    q, qw = g8.quantized(x), g8.quantized_kernels(w)
    y = g8.rows(q, qw, torch.tensor([50, 40], dtype=torch.int32).cuda(), F32).double()
    for g, (lo, hi) in enumerate(((0, 50), (50, 90))):
        xs, ws = x[lo:hi].double(), w[g].double()
        sx, sw = q.scales[lo:hi].double()[:, None], qw.scales[g].double()
        bound = (sw / 2 * xs.abs().sum(-1, keepdim=True) + sx / 2 * ws.abs().sum(0) + 500 * sx * sw / 4)
        size = xs.abs() @ ws.abs()
        assert ((y[lo:hi] - xs @ ws).abs() <= bound * 1.001 + 6 * 2.0**-24 * size).all()


def _layer(seed, t, d, e, k, f, p=2, dtype=BF16):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(t, d, generator=g).to(dtype).cuda()
    w, idx = torch.topk(torch.softmax(torch.randn(t, e, generator=g), -1), k, -1)
    up = (0.05 * torch.randn(e, d, f, p, generator=g)).to(dtype).cuda()
    down = (0.05 * torch.randn(e, f, d, generator=g)).to(dtype).cuda()
    return z, idx.int().cuda(), w.to(dtype).cuda(), up, down, g


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("t,d,e,k,f,p,extras", [
    (1, 64, 4, 2, 32, 2, False), (9, 200, 6, 3, 100, 2, True), (300, 256, 8, 2, 128, 1, True),
    (700, 136, 40, 4, 68, 2, False), (0, 64, 4, 2, 32, 2, False)])
def test_the_layer_is_its_steps(lib, t, d, e, k, f, p, extras, dtype):
    """experts_int8 against its steps, each by the public op that the other tests hold; picks
    outside the experts; and near the same layer in float arithmetic."""
    from bux_amd import grouped_int8 as g8, moe
    announce("int8 layer", t, d, e, k, f, p, extras, dtype)
    z, idx, w, up, down, g = _layer(t + d, t, d, e, k, f, p, dtype)
    if t > 2:
        idx[1, 0] = e + 3
        idx[2, k - 1] = -1
    ffn = moe.Ffn("swish") if p == 2 else moe.Ffn("relu2")
    ub = (0.1 * torch.randn(e, f, p, generator=g)).to(dtype).cuda() if extras else None
    db = (0.1 * torch.randn(e, d, generator=g)).to(dtype).cuda() if extras else None
    weights = moe.in_int8(up, down)
    y = moe.experts_int8(z, idx, w, weights, ffn, ub, db)
    m = t * k
    s = moe.sort_by_expert(idx.view(-1), e)
    x = g8.quantized(z, s.filled, s.order, k)
    row_w = moe.picked_weights(w, s.order)
    projected = g8.rows(x, weights.up, s.sizes, dtype,
                        bias=None if ub is None else ub.reshape(e, f * p))
    h = moe.weighted_units(ffn, projected.view(m, f, p), row_w, s.filled)
    rows = g8.rows(g8.quantized(h, s.filled), weights.down, s.sizes, dtype)
    if db is None:
        want = moe.sum_by_token(rows, s.inverse.view(t, k))
    else:
        want = moe.sum_by_token_biased(rows, s.inverse.view(t, k), db, s.offsets, row_w)
    assert torch.equal(y, want)


def test_the_layer_in_a_graph_and_repeated(lib):
    """A decode step captured once and replayed over new tokens and picks."""
    from bux_amd import moe
    z, idx, w, up, down, _ = _layer(1, 8, 256, 16, 4, 128)
    weights = moe.in_int8(up, down)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        moe.experts_int8(z, idx, w, weights)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = moe.experts_int8(z, idx, w, weights)
    for seed in (2, 3, 4):
        for old, new in zip((z, idx, w), _layer(seed, 8, 256, 16, 4, 128)):
            old.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        want = moe.experts_int8(z, idx, w, weights)
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_the_layer_with_a_norm_of_its_outputs(lib):
    from bux_amd import grouped_int8 as g8, moe
    z, idx, w, up, down, g = _layer(6, 50, 128, 8, 2, 64)
    scale = (1 + 0.1 * torch.randn(128, generator=g)).to(BF16).cuda()
    norm = moe.ExpertNorm("rmsnorm")
    weights = moe.in_int8(up, down)
    y = moe.experts_int8(z, idx, w, weights, norm=norm, norm_scale=scale)
    s = moe.sort_by_expert(idx.view(-1), 8)
    row_w = moe.picked_weights(w, s.order)
    projected = g8.rows(g8.quantized(z, s.filled, s.order, 2), weights.up, s.sizes)
    h = moe.weighted_units_int8(moe.Ffn(), projected.view(100, 64, 2), torch.ones_like(row_w), s.filled)
    rows = moe.expert_norm_forward(g8.rows(h, weights.down, s.sizes), s.offsets, norm, scale, None, row_w)
    assert torch.equal(y, moe.sum_by_token(rows, s.inverse.view(50, 2)))


def test_the_blocks_operators_together(lib):
    """A block's step as a program runs it: the norm with the residual, the router, the experts;
    their backward, the router's gradient added to the experts' and through the norm; and the
    same tokens served in 8-bit integers, near the training path's output."""
    from bux_amd import moe, norm as tnorm, router
    g = torch.Generator().manual_seed(21)
    t, d, e, k, f = 200, 256, 16, 4, 128
    x, res = (torch.randn(t, d, generator=g).to(BF16).cuda() for _ in range(2))
    scale = (1 + 0.1 * torch.randn(d, generator=g)).to(BF16).cuda()
    kernel = (0.05 * torch.randn(d, e, generator=g)).to(BF16).cuda()
    up = (0.05 * torch.randn(e, d, f, 2, generator=g)).to(BF16).cuda()
    down = (0.05 * torch.randn(e, f, d, generator=g)).to(BF16).cuda()
    dy = (0.1 * torch.randn(t, d, generator=g)).to(BF16).cuda()
    settings = moe.ExpertNorm("rmsnorm")
    n = tnorm.normed(x, settings, scale, residual=res)
    r = router.route(n.out, kernel, top_k=k, with_logits=True)
    y, saved = moe.experts_forward(n.out, r.idx, r.weights, up, down, fmt="compute")
    grads = moe.experts_backward(saved, dy, up, down, fmt="compute")
    rg = router.route_backward(n.out, kernel, r.idx, r.logits, grads["weights"], dz=grads["z"])
    ng = tnorm.normed_backward(rg.x, n.summed, n.stats, settings, scale, d_summed=dy)
    served = moe.experts_int8(n.out, r.idx, r.weights, moe.in_int8(up, down))
    # two roundings to 8 bits in a row (a 254th of a row's largest value, some 3 of its mean
    # square root, uniformly: 0.7% a factor) of four factors: within 3 percent in norm
    off = (served.double() - y.double()).norm() / y.double().norm()
    assert off < 0.03, float(off)
    # the whole step's gradient to x along a direction, against differences of the float64 block
    # with the picks held: bfloat16 roundings at every op bound it to a few percent
    def block(x, kernel):
        v = x.double() + res.double()
        h = v / (v.square().mean(-1, keepdim=True) + settings.eps).sqrt() * scale.double()
        s = torch.softmax(h @ kernel.double(), -1).gather(1, r.idx.long())
        s = s / s.sum(-1, keepdim=True)
        out = v.clone()  # the residual stream goes on
        for j in range(k):
            for q in range(e):
                at = (r.idx[:, j] == q).nonzero()[:, 0]
                p = (h[at] @ up[q].double().reshape(d, 2 * f)).view(-1, f, 2)
                u = p[..., 1] * torch.sigmoid(p[..., 1]) * p[..., 0]
                out[at] += s[at, j, None] * (u @ down[q].double())
        return float((out * dy.double()).sum())

    for which, grad, at in (("x", ng.x, x), ("kernel", rg.kernel, kernel)):
        v = torch.randn(at.shape, generator=g, dtype=torch.float64).cuda()
        step = 1e-4
        a = {"x": x.double(), "kernel": kernel.double()}
        up_, dn_ = dict(a), dict(a)
        up_[which], dn_[which] = a[which] + step * v, a[which] - step * v
        want = (block(**up_) - block(**dn_)) / (2 * step)
        got = float((grad.double() * v).sum())
        noise = float((grad.double() * v).square().sum().sqrt())
        assert abs(got - want) <= 0.02 * abs(want) + 0.05 * noise, (which, got, want)


def test_refusals(lib):
    from bux_amd import grouped_int8 as g8, moe
    x = _normal(1, 8, 64)
    w = _normal(2, 2, 64, 32)
    a, b = g8.quantized(x), g8.quantized_kernels(w)
    sz = torch.tensor([4, 4], dtype=torch.int32).cuda()
    with pytest.raises(TypeError, match="float16"):
        g8.quantized(x.half())
    with pytest.raises(ValueError, match="height"):
        g8.quantized(x, height=7)
    with pytest.raises(ValueError, match="index"):
        g8.quantized(x, index=sz.long())
    with pytest.raises(ValueError, match="index_div"):
        g8.quantized(x, index=sz, index_div=0)
    with pytest.raises(ValueError, match="contiguous"):
        g8.quantized(x.t())
    with pytest.raises(ValueError, match="matrix"):
        g8.quantized(x[0])
    with pytest.raises(ValueError, match="codes"):
        g8.rows(a, g8.quantized_kernels(_normal(3, 2, 200, 32)), sz)
    with pytest.raises(ValueError, match="multiple of 4"):
        g8.rows(a, g8.quantized_kernels(_normal(3, 2, 64, 30)), sz)
    with pytest.raises(ValueError, match="int32"):
        g8.rows(a, b, sz.long())
    with pytest.raises(ValueError, match=r"\(2, 32\)"):
        g8.rows(a, b, sz, bias=_normal(4, 2, 31))
    with pytest.raises(TypeError, match="float16"):
        g8.rows(a, b, sz, torch.float16)
    with pytest.raises(ValueError, match="in_int8"):
        moe.in_int8(_normal(1, 2, 64, 32, 2), _normal(1, 2, 64, 64))
    for d, f in ((64, 6), (132, 68)):  # the token sums take whole eights of columns
        with pytest.raises(ValueError, match="multiple of 8"):
            moe.in_int8(_normal(1, 2, d, f, 2), _normal(1, 2, f, d))
    weights = moe.in_int8(_normal(1, 2, 64, 32, 2), _normal(1, 2, 32, 64))
    idx = torch.zeros(8, 1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="tokens"):
        moe.experts_int8(_normal(1, 8, 60), idx, x[:, :1].contiguous(), weights)
    with pytest.raises(ValueError, match="weights"):
        moe.experts_int8(x, idx, x[:, :2].contiguous(), weights)
