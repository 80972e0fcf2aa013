"""The router's backward holds the logits' gradient G in float32 in its products.

Sums that cancel show it: pairs of logits (for dx) and of tokens (for d_kernel) whose gradients
differ by some 2^-20 of themselves, against columns that are each other's negatives. A product of
G's parts and a bfloat16 is exact; a sum adds a unit in the last place, 2^-23 of the terms'
magnitudes, for each of 3 parts a term. (In two parts of 8 bits G itself is off by up to 2^-17.)
"""

import pytest
import torch

from _util import announce

pytestmark = pytest.mark.gpu

BF16, F64 = torch.bfloat16, torch.float64
HALF_STEP = 2.0 ** -8
UNIT = 2.0 ** -23
PARTS = 3


def _within(got, want, tolerance, what):
    off = (got.double() - want).abs() / tolerance
    assert off.max() <= 1, (what, float(off.max()))


@pytest.mark.parametrize("magnitude", [1.0, 1e-30, 1e30])
@pytest.mark.parametrize("seed", range(4))
def test_sums_that_cancel(lib, seed, magnitude):
    from bux_amd import router
    announce("route backward, sums that cancel", seed, magnitude)
    g = torch.Generator().manual_seed(seed)
    t, n, d = 2, 2, 256
    G = (1 + torch.rand(1, 1, generator=g, dtype=F64)
         * (1 + torch.randn(t, n, generator=g, dtype=F64) * 2.0 ** -19)).float() * magnitude
    x = torch.randn(1, d, generator=g).to(BF16)
    x = torch.cat([x, -x])
    kernel = torch.randn(d, 1, generator=g).to(BF16)
    kernel = torch.cat([kernel, -kernel], 1)
    v = {"logits": torch.randn(t, n, generator=g), "d_logits": G, "x": x, "kernel": kernel,
         "idx": torch.zeros(t, 1, dtype=torch.int32), "d_weights": torch.zeros(t, 1, dtype=BF16)}
    v = {key: a.cuda() for key, a in v.items()}
    got = router.route_backward(v["x"], v["kernel"], v["idx"], v["logits"], v["d_weights"],
                                normalize_top_k=False, d_logits=v["d_logits"])
    G, x, kernel = (v[key].double() for key in ("d_logits", "x", "kernel"))
    dx, size = G @ kernel.t().contiguous(), G.abs() @ kernel.abs().t().contiguous()
    _within(got.x, dx, HALF_STEP * dx.abs() + PARTS * n * UNIT * size, "x")
    dk, size = x.t().contiguous() @ G, x.abs().t().contiguous() @ G.abs()
    _within(got.kernel, dk, HALF_STEP * dk.abs() + PARTS * t * UNIT * size, "kernel")


def test_the_whole_range_of_float32(lib):
    """The largest finite gradients and those far below 1 pass as they are."""
    from bux_amd import router
    big = torch.finfo(torch.float32).max
    values = torch.tensor([[big, -big], [2.0 ** -100, 1.0], [2.0 ** 127, 3.0 * 2.0 ** -90]])
    for token in values:
        G = token.view(1, 2).cuda()
        x = torch.full((1, 16), 0.5, dtype=BF16, device="cuda")
        kernel = torch.full((16, 2), 0.25, dtype=BF16, device="cuda")
        kernel[:, 1] = 0
        got = router.route_backward(x, kernel, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                                    torch.zeros(1, 2, device="cuda"),
                                    torch.zeros(1, 1, dtype=BF16, device="cuda"),
                                    normalize_top_k=False, d_logits=G)
        assert torch.equal(got.x, (G[:, :1] * 0.25).to(BF16).expand(1, 16))
        assert torch.equal(got.kernel, (G * 0.5).to(BF16).expand(16, 2))
        assert torch.equal(got.bias, G[0])
