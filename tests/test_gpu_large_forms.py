"""The forms that the largest calls of the norm's and the router's backward run, by the checks of
the other tests: waves of 64 tokens (above 128 logits, where their workgroups fill the chip), and
rows of 8 waves whose workgroups take several rows, the next one on its way through LDS."""

import pytest
import torch

import test_gpu_norm as norms
import test_gpu_route_backward as routes
from _util import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,d,n,scored,k,router,normalize,extras", [
    (1090, 8192, 160, 160, 8, "softmax", True, {"dz": True}),
    (1090, 8192, 160, 160, 8, "sigmoid", True, {"scores": True}),
    (1055, 8176, 250, 240, 4, "softmax", False, {"dz": True, "sinks": True, "logits": True}),
    (2049, 4096, 1000, 1000, 16, "sqrtsoftplus", True, {"dz": True, "scores": True}),
])
def test_route_backward_of_many_workgroups(lib, t, d, n, scored, k, router, normalize, extras):
    announce("route backward", t, d, n, router, extras)
    assert n > 128 and -(-t // 64) * -(-d // 512) >= 256
    routes._compare(routes._inputs(t, d, n, scored, k, seed=t + n, **extras), scored, router, normalize,
                    1.0, 2.5)


@pytest.mark.parametrize("name", ["rms", "layer", "layer zero-centered scale input"])
@pytest.mark.parametrize("m,d", [(600, 7168), (530, 6152), (521, 12288)])
def test_norm_of_wide_rows_in_turns(lib, m, d, name):
    norms.test_forward_and_backward(lib, m, d, name, torch.bfloat16)


@pytest.mark.parametrize("m,d", [(600, 7168), (521, 12288)])
def test_norm_of_wide_rows_at_any_alignment(lib, m, d):
    norms.test_the_same_bits_at_any_alignment(lib, m, d)
