"""8-bit products whose sizes, which lie on the device, put rows of a group past a's: they are
products of 0 (with the group's bias), by either kernel, and read nothing past a or its scales.
Exact, as the products are."""

import pytest
import torch

from _util import announce

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _operands(m, n, k, groups, seed):
    """a, b and their codes row-major; a's buffers end where its rows do, in one of NaN scales."""
    from bux_amd import grouped_int8 as g8
    g = torch.Generator().manual_seed(seed)
    out = []
    for lead, rows in (((), m), ((groups,), n)):
        codes = torch.randint(-127, 128, (*lead, rows, k), generator=g, dtype=torch.int8)
        tiled = codes.view(*lead, rows, k // 64, 64).transpose(-3, -2).contiguous().cuda()
        scales = torch.rand(*lead, rows, generator=g) * 0.01 + 1e-4
        held = torch.full((scales.numel() + 512,), float("nan"), device="cuda")
        held[:scales.numel()] = scales.view(-1).cuda()
        out.append((g8.Int8(tiled, held[:scales.numel()].view(scales.shape)), codes, scales))
    return out


# groups, sizes, a's rows, y's height: few rows a group, then many
CASES = [
    (4, [3, 5, 40, 9], 20, 70),       # the third group's rows end past a's
    (40, [1] * 39 + [2**31 - 1], 50, 300),  # the last one's take all of y
    (40, [0] * 39 + [100], 1, 100),
    (3, [4, 4, 4], 0, 30),            # no rows at all
    (3, [0, 0, 0], 0, 5),
    (2, [100, 150], 180, 300),        # and past the line to the other kernel
    (2, [10, 300], 40, 256),
]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("biased", [False, True], ids=["", "biased"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-{c[2]}-{c[3]}")
def test_rows_that_sizes_put_past_the_operand(lib, case, biased, dtype):
    from bux_amd import grouped_int8 as g8
    groups, sizes, m, height = case
    announce("int8 products past the rows", case, biased, dtype)
    n, k = 72, 256
    (a, ac, sa), (b, bc, sb) = _operands(m, n, k, groups, seed=m + height)
    bias = torch.randn(groups, n, generator=torch.Generator().manual_seed(1)).to(dtype) if biased else None
    y = g8.rows(a, b, torch.tensor(sizes, dtype=torch.int32).cuda(), dtype, height,
                bias=None if bias is None else bias.cuda())
    want = torch.zeros(height, n)
    row = 0
    for g, size in enumerate(sizes):
        end = min(row + size, max(m, height))
        for i in range(row, min(end, height)):
            if i < m:
                s = (ac[i].double() * bc[g].double()).sum(-1)
                want[i] = s.float() * (sa[i] * sb[g])
            if biased:
                want[i] += bias[g].float()
        row = end
    assert torch.equal(y.cpu(), want.to(dtype)), (y.cpu() != want.to(dtype)).nonzero()[:5]
