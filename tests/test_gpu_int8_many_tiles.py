"""8-bit products whose workgroups take several tiles one after another, and those of operands
past 2 GiB: exact, as the others are.

A tile's scales lie in one of two places that a workgroup's tiles take in turn, while the next
tile's first steps load; K of 128 is two steps, fewer than those loads run ahead. Groups of a row, of
half tiles, of whole ones and of one row more, empty ones, and rows past them all, in every order."""

import pytest
import torch

from _util import announce

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _codes(gen, *shape):
    return torch.randint(-127, 128, shape, generator=gen, dtype=torch.int8, device="cuda")


def _scales(gen, *shape):
    return torch.rand(*shape, generator=gen, device="cuda") * 0.01 + 1e-4


def _row_major(values):
    """(..., K / 64, rows, 64) codes as (..., rows, K)."""
    v = values.transpose(-3, -2)
    return v.reshape(*v.shape[:-2], -1)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("biased", [False, True], ids=["", "biased"])
@pytest.mark.parametrize("k,n", [(128, 1028), (384, 772), (640, 512)])
def test_workgroups_of_many_tiles(lib, k, n, biased, dtype):
    from bux_amd import grouped_int8 as g8
    announce("int8 products of many tiles", k, n, biased, dtype)
    sizes = [1, 300, 0, 128, 129, 256, 600, 5, 257, 511, 0, 0, 127, 64, 1000, 385] * 12 + [90]
    filled = sum(sizes)
    m, height = filled + 700, filled + 1100
    # tiles of 256 rows by 256 columns, at least this many; a workgroup a CU
    tiles = (sum(-(-s // 256) for s in sizes) + 1100 // 256) * -(-n // 256)
    assert tiles > 2 * torch.cuda.get_device_properties(0).multi_processor_count
    assert m > 16 * len(sizes)
    gen = torch.Generator(device="cuda").manual_seed(k + n)
    a = g8.Int8(_codes(gen, k // 64, m, 64), _scales(gen, m))
    b = g8.Int8(_codes(gen, len(sizes), k // 64, n, 64), _scales(gen, len(sizes), n))
    bias = torch.randn(len(sizes), n, generator=gen, device="cuda").to(dtype) if biased else None
    y = g8.rows(a, b, torch.tensor(sizes, dtype=torch.int32).cuda(), dtype, height, bias=bias)
    ac, bc = _row_major(a.values), _row_major(b.values)
    row = 0
    for g, size in enumerate(sizes):
        at = slice(row, row + size)
        sums = (ac[at].double() @ bc[g].double().t()).float()  # below 2^24, or rounded as the op does
        want = sums * (a.scales[at, None] * b.scales[g])
        if biased:
            want = want + bias[g].float()
        assert torch.equal(y[at], want.to(dtype)), (g, size)
        row += size
    assert (y[row:] == 0).all()


def _narrow(a, b, sizes, rows, columns, dtype):
    """The product of a slice of one group's rows and columns."""
    from bux_amd import grouped_int8 as g8
    return g8.rows(g8.Int8(a.values[:, rows].contiguous(), a.scales[rows].contiguous()),
                   g8.Int8(b.values[..., columns, :].contiguous(), b.scales[:, columns].contiguous()),
                   sizes, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_tokens_past_2_gib(lib, dtype):
    """A long prompt's rows: every row as in a product of some thousands of them."""
    from bux_amd import grouped_int8 as g8
    announce("int8 products, a past 2 GiB", dtype)
    m, k, n = 300_000, 7168, 68
    gen = torch.Generator(device="cuda").manual_seed(3)
    a = g8.Int8(_codes(gen, k // 64, m, 64), _scales(gen, m))
    b = g8.Int8(_codes(gen, 3, k // 64, n, 64), _scales(gen, 3, n))
    assert a.values.numel() > 2**31
    sizes = [100_001, 130_000, m - 230_001 - 999]
    y = g8.rows(a, b, torch.tensor(sizes, dtype=torch.int32).cuda(), dtype)
    row = 0
    for g, size in enumerate(sizes):
        own = g8.Int8(b.values[g:g + 1].contiguous(), b.scales[g:g + 1].contiguous())
        for lo, hi in ((row, row + 700), (row + size // 2, row + size // 2 + 700), (row + size - 700, row + size)):
            part = _narrow(a, own, torch.tensor([hi - lo], dtype=torch.int32).cuda(), slice(lo, hi),
                           slice(0, n), dtype)
            assert (part != 0).any(1).all() and torch.equal(y[lo:hi], part), (g, lo)
        row += size
    assert (y[row:] == 0).all()


@pytest.mark.parametrize("biased", [False, True], ids=["", "biased"])
def test_kernels_past_2_gib(lib, biased):
    from bux_amd import grouped_int8 as g8
    announce("int8 products, b past 2 GiB", biased)
    m, k, n = 150, 131_072, 16_644
    gen = torch.Generator(device="cuda").manual_seed(4)
    a = g8.Int8(_codes(gen, k // 64, m, 64), _scales(gen, m))
    b = g8.Int8(_codes(gen, 1, k // 64, n, 64), _scales(gen, 1, n))
    assert b.values.numel() > 2**31
    bias = torch.randn(1, n, generator=gen, device="cuda") if biased else None
    sizes = torch.tensor([m], dtype=torch.int32).cuda()
    y = g8.rows(a, b, sizes, F32, bias=bias)
    for lo in (0, 8192, n - 260):
        part = _narrow(a, b, sizes, slice(0, m), slice(lo, lo + 260), F32)
        if biased:
            part = part + bias[:, lo:lo + 260]
        assert (part != 0).any(0).all() and torch.equal(y[:, lo:lo + 260], part), lo
