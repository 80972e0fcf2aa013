"""Dense bfloat16 products whose operands reach past what the large tiles' and the few rows' kernels
address (32-bit offsets): a head's kernel of over 2^30 elements, a contraction over as many. The
128 x 128 tiles take them. Columns at both ends and where the operand's bytes pass 2^31, against the
formulas in float64, within bounds counted beforehand (tests/_dense.py)."""

import pytest
import torch

from _dense import BF16, F64, V
from _util import announce

pytestmark = pytest.mark.gpu


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=BF16)


def _v(t):
    return V(t.to(F64))


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("transposed", [False, True], ids=["", "transposed"])
def test_a_wide_head(lib, transposed, m):
    from bux_amd import dense

    k, n = 7168, 151936
    g = torch.Generator(device="cuda").manual_seed(m)
    x, w = _randn(g, m, k), _randn(g, *((n, k) if transposed else (k, n)))
    announce("dense wide head", m, transposed)
    got = dense.product(x, w, transposed=transposed).out
    line = 2 ** 30 // k
    cols = torch.cat([torch.arange(64), torch.arange(line - 32, line + 32), torch.arange(n - 64, n)])
    cols = cols.cuda()
    part = w[cols].t() if transposed else w[:, cols]
    (_v(x) @ _v(part.contiguous())).rounded(BF16).holds(got[:, cols], "out")
    dy = _randn(g, m, n)
    dx = dense.product_backward(dy, x, w, transposed=transposed).x
    # every column of w, some of its rows
    rows = torch.cat([torch.arange(16), torch.arange(k - 16, k)]).cuda()
    part = (w[:, rows] if transposed else w[rows].t()).contiguous()
    (_v(dy) @ _v(part)).rounded(BF16).holds(dx[:, rows], "dx")


@pytest.mark.parametrize("wide", ["x", "dy"])
def test_a_contraction_over_many_rows(lib, wide):
    from bux_amd import dense

    m, k, n = 65608, 16384, 264
    g = torch.Generator(device="cuda").manual_seed(3)
    x, dy = _randn(g, m, k), _randn(g, m, n)
    announce("dense long contraction", wide)
    dw = dense.weight_grad(x, dy) if wide == "x" else dense.weight_grad(dy, x).t()
    cols = torch.cat([torch.arange(32), torch.arange(k // 2 - 16, k // 2 + 16),
                      torch.arange(k - 32, k)]).cuda()
    (_v(x[:, cols].contiguous()).t() @ _v(dy)).rounded(BF16).holds(dw[cols], "dw")
