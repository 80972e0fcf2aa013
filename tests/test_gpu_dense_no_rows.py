"""Dense products of no rows, forward and backward, with an activation and without: empty rows, and
gradients of 0 to what has no rows."""

import pytest
import torch

from _util import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bias", [False, True], ids=["", "bias"])
@pytest.mark.parametrize("activation", [None, "swish", "gelu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("transposed", [False, True], ids=["", "transposed"])
def test_product(lib, transposed, dtype, activation, bias):
    from bux_amd import dense

    new = dict(dtype=dtype, device="cuda")
    x, w = torch.zeros(2, 0, 96, **new), torch.ones(*((80, 96) if transposed else (96, 80)), **new)
    announce("dense no rows", dtype, activation, bias, transposed)
    got = dense.product(x, w, torch.ones(80, **new) if bias else None, activation,
                        x.new_zeros(2, 0, 80), transposed, with_product=activation is not None)
    assert got.out.shape == (2, 0, 80)
    grads = dense.product_backward(x.new_zeros(2, 0, 80), x, w, activation, got.product, transposed,
                                   bias)
    assert grads.x.shape == x.shape and grads.w.shape == w.shape and not grads.w.any()
    if bias:
        assert grads.bias.shape == (80,) and not grads.bias.any()
    else:
        assert grads.bias is None
