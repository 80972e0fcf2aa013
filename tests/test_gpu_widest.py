"""Grouped products of the widest outputs that their stores hold: each column is what the
same column gives in a narrow product, to the bit, in every row."""

import pytest
import torch

from _util import announce

pytestmark = pytest.mark.gpu

N = (1 << 22) - 4  # a tile's 256 rows of it are just below 2 GiB of bfloat16
COLUMNS = [0, 4, N // 3 // 4 * 4, N // 2, N - 256, N - 4]


def _narrow(values, axis):
    """The operand's rows from each of COLUMNS on, four at a time."""
    at = torch.cat([torch.arange(c, c + 4) for c in COLUMNS]).cuda()
    return values.index_select(axis, at).contiguous(), at


@pytest.mark.parametrize("height", [256, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_8_bit_products(lib, height, dtype):
    from bux_amd import grouped_int8 as g8
    announce("widest int8", height, dtype)
    m, k = 256, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    a = g8.Int8(torch.randint(-127, 128, (2, m, 64), generator=g, dtype=torch.int8, device="cuda"),
                torch.rand(m, generator=g, device="cuda"))
    b = g8.Int8(torch.randint(-127, 128, (1, 2, N, 64), generator=g, dtype=torch.int8, device="cuda"),
                torch.rand(1, N, generator=g, device="cuda"))
    sizes = torch.tensor([m], dtype=torch.int32, device="cuda")
    y = g8.rows(a, b, sizes, dtype, height)
    values, at = _narrow(b.values, 2)
    want = g8.rows(a, g8.Int8(values, _narrow(b.scales, 1)[0]), sizes, dtype, height)
    assert (want != 0).any(1)[:m].all()
    assert torch.equal(y[:, at], want)
    assert (y[m:] == 0).all()


def test_mxfp8_products(lib):
    from bux_amd import grouped_mxfp8
    announce("widest MXFP8")
    m, k, height = 256, 128, 257
    g = torch.Generator(device="cuda").manual_seed(2)

    def operand(*lead, rows):
        v = torch.randint(0, 0x70, (*lead, 2, rows, 64), generator=g, dtype=torch.uint8, device="cuda")
        s = torch.randint(120, 126, (*lead, 1, rows, 4), generator=g, dtype=torch.uint8, device="cuda")
        return grouped_mxfp8.Tiled(v, s)

    a, b = operand(rows=m), operand(1, rows=N)
    sizes = torch.tensor([m], dtype=torch.int32, device="cuda")
    y = grouped_mxfp8.rows(a, b, sizes, height=height)
    values, at = _narrow(b.values, 2)
    want = grouped_mxfp8.rows(a, grouped_mxfp8.Tiled(values, _narrow(b.scales, 2)[0]), sizes, height=height)
    assert (want != 0).any(1)[:m].all()
    assert torch.equal(y[:, at], want) and (y[m:] == 0).all()
