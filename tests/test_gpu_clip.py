"""The gradients' global norm and their clipping (bux_amd.clip) against float64.

The norm: float64 sums, one rounding to float32, 2^-24 of it (and 1e-12 for the sums). A clipped
value: the factor's rounding to float32, the product's, then its type's: eps / 2 + 2^-23."""

import math

import pytest
import torch

from _util import announce

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def _grads(g, shapes):
    return [(s * torch.randn(*shape, generator=g)).to(dt).cuda() for shape, dt, s in shapes]


LISTS = {
    "one value": [((1,), F32, 1.0)],
    "seven": [((7,), BF16, 1.0)],
    "a piece and one": [((8193,), BF16, 1.0), ((8191,), F32, 2.0)],
    "mixed": [((3, 5, 7), BF16, 0.1), ((1000, 33), F32, 0.01), ((0,), F32, 1.0), ((2,), BF16, 9.0),
              ((70000,), BF16, 0.02)],
    "many": [((17 + i, 3), F32 if i % 3 else BF16, 0.1 * i) for i in range(150)],
    "all empty": [((0,), BF16, 1.0), ((0, 4), F32, 1.0)],
    "large": [((40_000_003,), BF16, 1e-3), ((5_000_001,), F32, 1e-3)],
}


@pytest.mark.parametrize("name", LISTS)
@pytest.mark.parametrize("in_place", [False, True], ids=["", "in place"])
def test_clipped(lib, name, in_place):
    from bux_amd import clip

    g = torch.Generator().manual_seed(1)
    grads = _grads(g, LISTS[name])
    want = [x.cpu().to(F64) for x in grads]
    norm = math.sqrt(sum(x.square().sum().item() for x in want))
    announce("clip", name, in_place)
    alone = clip.global_norm(grads)
    assert alone.dtype == F32 and alone.shape == ()
    assert abs(alone.item() - norm) <= (2.0 ** -24 + 1e-12) * norm
    for most in (0.3 * norm or 1.0, 2 * norm or 1.0):
        at = [x.clone() for x in grads]
        r = clip.clipped(at, most, in_place)
        assert torch.equal(r.norm, alone)
        factor = 1.0 if norm <= most else float(torch.tensor(most, dtype=F32)) / norm
        for x, w, o, a in zip(grads, want, r.grads, at):
            assert o.shape == x.shape and o.dtype == x.dtype
            assert (o.data_ptr() == a.data_ptr()) == in_place or not x.numel()
            if factor == 1.0:
                assert torch.equal(o, x)
                continue
            off = (o.cpu().to(F64) - w * factor).abs()
            assert (off <= (torch.finfo(x.dtype).eps / 2 + 2.0 ** -23) * (w * factor).abs()).all()
            assert in_place or torch.equal(a, x)


def test_squares_outside_float32(lib):
    from bux_amd import clip

    for value in (1e30, 1e-30):
        for dt in (BF16, F32):
            x = torch.full((100, 100), value, dtype=dt, device="cuda")
            want = 100 * x[0, 0].double().item()
            assert abs(clip.global_norm([x]).item() - want) <= 2.0 ** -23 * want
            r = clip.clipped([x], want / 4).grads[0].double()
            assert ((r - x.double() / 4).abs() <= torch.finfo(dt).eps * x.double().abs()).all()


def test_infinities_and_nan(lib):
    from bux_amd import clip

    x = torch.ones(9000, dtype=BF16, device="cuda")
    y = torch.ones(5, device="cuda")
    x[8999] = float("inf")
    r = clip.clipped([x, y], 1.0)
    assert r.norm.isinf() and not r.grads[1].any() and not r.grads[0][:-1].any()
    assert r.grads[0][-1].isnan()
    x[8999] = float("nan")
    r = clip.clipped([x, y], 1.0)
    assert r.norm.isnan() and all(o.isnan().all() for o in r.grads)
    zero = clip.clipped([torch.zeros(10, device="cuda")], 1.0)
    assert zero.norm.item() == 0 and not zero.grads[0].any()


def test_odd_elements_and_their_neighbours(lib):
    """Tensors that begin at any element, in place: nothing beside them is read or written."""
    from bux_amd import clip

    for dt in (BF16, F32):
        for n in (1, 8, 4099, 8192, 20001):
            flat = torch.full((n + 6,), float("nan"), dtype=dt, device="cuda")
            flat[3:3 + n] = 2.0
            announce("clip odd", dt, n)
            r = clip.clipped([flat[3:3 + n]], 1.0, in_place=True)
            assert abs(r.norm.item() - 2 * math.sqrt(n)) <= 2.0 ** -23 * 2 * math.sqrt(n)
            assert flat[:3].isnan().all() and flat[3 + n:].isnan().all()
            assert not flat[3:3 + n].isnan().any()


def test_a_tensor_twice(lib):
    from bux_amd import clip

    x = torch.full((50,), 3.0, device="cuda")
    assert abs(clip.global_norm([x, x]).item() - 30.0) <= 2.0 ** -19
    r = clip.clipped([x, x], 15.0)
    assert torch.equal(r.grads[0], r.grads[1]) and torch.allclose(r.grads[0], x / 2)
    with pytest.raises(ValueError, match="twice"):
        clip.clipped([x, x], 15.0, in_place=True)
    with pytest.raises(ValueError, match="twice"):  # a part of another's memory
        clip.clipped([x[40:], x[10:41], x[:10]], 15.0, in_place=True)
    apart = clip.clipped([x[25:], x[:25]], 3.0, in_place=True)
    assert torch.equal(torch.cat([apart.grads[1], apart.grads[0]]), x)


def test_captured(lib):
    from bux_amd import clip

    g = torch.Generator().manual_seed(2)
    static = _grads(g, LISTS["mixed"])
    clip.clipped(static, 0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    announce("clip graph")
    with torch.cuda.graph(graph):
        r = clip.clipped(static, 0.5)
    for _ in range(3):
        fresh = _grads(g, LISTS["mixed"])
        for a, b in zip(static, fresh):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = clip.clipped(fresh, 0.5)
        torch.cuda.synchronize()
        assert torch.equal(r.norm, want.norm)
        assert all(torch.equal(a, b) for a, b in zip(r.grads, want.grads))


def test_refusals(lib):
    from bux_amd import clip

    x = torch.ones(4, 4, device="cuda")
    with pytest.raises(ValueError, match="no gradients"):
        clip.clipped([], 1.0)
    with pytest.raises(ValueError, match="no gradients"):
        clip.global_norm([])
    for most in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            clip.clipped([x], most)
    with pytest.raises(TypeError, match="float16"):
        clip.clipped([x, x.half()], 1.0)
    with pytest.raises(ValueError, match="contiguous"):
        clip.clipped([x.t().contiguous().t()[:, :2]], 1.0)
    with pytest.raises(ValueError, match="on cpu"):
        clip.clipped([x, x.cpu()], 1.0)
