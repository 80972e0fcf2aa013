"""The global norm of a step's gradients on MI355X, and their clipping by it: of the experts'
(`moe.experts_backward`), the router's (`router.route_backward`), the norms'
(`norm.normed_backward`) and the dense block's (`mlp.feed_forward_backward`) alike, bfloat16 and
float32 in one list.
"""

import ctypes
from typing import NamedTuple, Sequence

import torch

from bux_amd import _lib
from bux_amd.kernels import lib, on_device, ptr, require, stream, workspace


class Clipped(NamedTuple):
    """What `clipped` returns."""

    grads: list[torch.Tensor]  # each gradient's shape and dtype
    norm: torch.Tensor  # float32 scalar: the global norm before the clipping


_DTYPES = {torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}


def _list(name: str, grads: Sequence[torch.Tensor], outs: Sequence[torch.Tensor] | None):
    """The gradients as ``bux_gradient``s, which are 4 words each."""
    words = []
    device = grads[0].get_device()
    for g, out in zip(grads, outs or grads):
        dtype = _DTYPES.get(g.dtype)
        if dtype is None:
            raise TypeError(f"{name}: gradients are bfloat16 or float32, not {g.dtype}")
        if g.get_device() != device:
            raise ValueError(f"{name}: a gradient on {g.device} beside {grads[0].device}")
        words += (g.data_ptr(), 0 if outs is None else out.data_ptr(), g.numel(), dtype)
    return (ctypes.c_int64 * len(words))(*words)


def _run(name: str, grads: Sequence[torch.Tensor], outs, max_norm: float) -> torch.Tensor:
    dev = grads[0].device
    norm = torch.empty((), dtype=torch.float32, device=dev)
    ws = workspace(lib().bux_clip_workspace_size(len(grads)), dev)
    _lib.check(lib().bux_clip(_list(name, grads, outs), len(grads), max_norm, ptr(norm), ptr(ws),
                              ws.numel(), stream()))
    return norm


def global_norm(grads: Sequence[torch.Tensor]) -> torch.Tensor:
    """Return ``(sum over all gradients of g^2)^(1/2)``, a float32 scalar on their GPU, added in
    float64 in a fixed order."""
    if not grads:
        raise ValueError("global_norm: no gradients")
    require(*grads)
    with on_device(grads[0]):
        return _run("global_norm", grads, None, 0.0)


def clipped(grads: Sequence[torch.Tensor], max_norm: float, in_place: bool = False) -> Clipped:
    """Return the gradients times ``min(1, max_norm / norm)`` and their `global_norm`; with
    `in_place` in the gradients' own memory. The factor and the products are float64's, rounded
    once to float32 and from there to bfloat16; the factor is of the float64 norm, also where
    the norm returned overflows float32. An infinite gradient scales by 0 (and becomes a NaN), a NaN
    makes every gradient NaN; with an infinite `max_norm` they stay as they are. The same tensor
    twice in one list counts twice (in place it is refused)."""
    if not grads:
        raise ValueError("clipped: no gradients")
    if not max_norm > 0:
        raise ValueError(f"clipped: max_norm {max_norm} is not above 0")
    require(*grads)
    if in_place:
        spans = sorted((g.data_ptr(), g.numel() * g.element_size()) for g in grads if g.numel())
        if any(a + size > b for (a, size), (b, _) in zip(spans, spans[1:])):
            raise ValueError("clipped: the same memory twice in one list, in place")
    with on_device(grads[0]):
        outs = list(grads) if in_place else [torch.empty_like(g) for g in grads]
        return Clipped(outs, _run("clipped", grads, outs, float(max_norm)))
