"""The clipping's factor, max_norm / norm (bux_amd.clip), against float64.

A float32 value is off by its one rounding, 2^-24, and the factor's and the norm's own in float64
(2^-50 covers them); a bfloat16 one goes through float32: 2^-8 + 2^-24. Results are normal numbers of
their type."""

import math

import pytest
import torch

from _util import announce

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
OFF = {F32: 2.0 ** -24 + 2.0 ** -50, BF16: 2.0 ** -8 + 2.0 ** -24 + 2.0 ** -50}


def _holds(grads, most, in_place):
    from bux_amd import clip

    want = [x.to(F64) for x in grads]
    norm = math.sqrt(sum(w.square().sum().item() for w in want))
    got = clip.clipped([x.clone() for x in grads], most, in_place)
    for w, o in zip(want, got.grads):
        exact = w * (float(torch.tensor(most, dtype=F32)) / norm)
        assert ((o.to(F64) - exact).abs() <= OFF[o.dtype] * exact.abs()).all(), (most, norm)


# values about `scale`, a limit: an ordinary one, and factors below float32's least normal number,
# 2^-126, and below its least number at all
@pytest.mark.parametrize("in_place", [False, True], ids=["", "in place"])
@pytest.mark.parametrize("scale, most", [(1e-2, 1.0), (3.0, 0.1), (1e37, 1.0), (1e37, 1e-3),
                                         (2e37, 1e-7)], ids=str)
def test_values_of_one_factor(lib, scale, most, in_place):
    g = torch.Generator().manual_seed(4)
    # magnitudes from 1 to 3 times the scale: no result is subnormal
    grads = [(scale * (1 + 2 * torch.rand(n, generator=g, dtype=F64))
              * torch.where(torch.rand(n, generator=g) < 0.5, -1.0, 1.0)).to(dt).cuda()
             for n, dt in ((70001, F32), (50003, BF16), (8192, F32), (16384, BF16), (3, F32))]
    announce("clip factor", scale, most, in_place)
    _holds(grads, most, in_place)


def test_a_norm_past_float32(lib):
    """The norm that is returned is float32's infinity; the gradients are scaled by the finite one."""
    from bux_amd import clip

    x = torch.full((10000,), 3e38, device="cuda")
    r = clip.clipped([x], 1.0)
    assert r.norm.isinf()
    assert ((r.grads[0].double() - 0.01).abs() <= 0.01 * (2.0 ** -24 + 2.0 ** -50)).all()


def test_no_limit(lib):
    """An infinite max_norm leaves the gradients as they are, whatever their norm."""
    from bux_amd import clip

    x = torch.tensor([1.0, -2.0, float("inf"), 0.1], device="cuda")
    for dt in (F32, BF16):
        for values in (x[:2], x):
            r = clip.clipped([values.to(dt)], float("inf"))
            assert torch.equal(r.grads[0], values.to(dt))
