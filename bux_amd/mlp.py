"""The dense feed-forward block on MI355X, gated or plain, and its backward: a model's ``mlp``
and ``gated_mlp`` layers (src/bux/architecture/layers/mlp.py:20-35), a shared expert beside the
routed ones, with the activation settings of `moe.Ffn`.

The up and gate projections, the activation and their product are one kernel (the up product's
epilogue); the down product adds its bias and the residual in its own. In the backward the down
product's gradient to the units goes through the activation's in its epilogue. bfloat16 or
float32: float32 sums and activation, one rounding of each output, of the units and of the
projections' gradient between the products.
"""

import ctypes
from typing import NamedTuple

import torch

from bux_amd import _lib
from bux_amd.dense import is_f32, room, rows_into, rows_of, shaped, slope, weight_grad
from bux_amd.kernels import lib, on_device, ptr, require, stream
from bux_amd.moe import Ffn
from bux_amd.spans import span


class Saved(NamedTuple):
    """What `feed_forward_backward` takes of the forward."""

    x: torch.Tensor  # the rows (..., d)
    projected: torch.Tensor  # x up + up_bias, before the activation (..., f, p)
    h: torch.Tensor  # the units (..., f)
    # bfloat16: int8, projected's next 8 bits (..., f, p), which keep the activation's gradient
    # from a second rounding beside its own; None (float32, or left out): from projected alone
    low: torch.Tensor | None = None


class FeedForward(NamedTuple):
    """What `feed_forward` returns."""

    out: torch.Tensor  # (..., d), x's dtype
    saved: Saved | None  # with `keep`


class FeedForwardGrads(NamedTuple):
    """What `feed_forward_backward` returns. (The residual's gradient is dy.)"""

    x: torch.Tensor  # x's shape
    up: torch.Tensor  # (d, f, p)
    down: torch.Tensor  # (f, d)
    up_bias: torch.Tensor | None  # (f, p), None if not asked for
    down_bias: torch.Tensor | None  # (d,)


def _kernels(name: str, up: torch.Tensor, down: torch.Tensor) -> tuple[int, int, int]:
    """(d, f, p) of the kernels up (d, f, p) and down (f, d)."""
    if up.dim() != 3 or up.shape[2] not in (1, 2) or up.numel() == 0:
        raise ValueError(f"{name}: up is (d, f, 2) or (d, f, 1), not {tuple(up.shape)}")
    d, f, p = up.shape
    shaped(name, "down", down, f, d)
    return d, f, p


def feed_forward(x: torch.Tensor, up: torch.Tensor, down: torch.Tensor, ffn: Ffn = Ffn(),
                 up_bias: torch.Tensor | None = None, down_bias: torch.Tensor | None = None,
                 residual: torch.Tensor | None = None, keep: bool = True) -> FeedForward:
    """Return ``h down + down_bias + residual`` with ``h = act(gate) (up + offset)`` of ``x up +
    up_bias`` for the rows x (..., d): up (d, f, 2), [..., 0] up and [..., 1] gate, or (d, f, 1)
    for a plain block, ``h = act(up)``; down (f, d); up_bias (f, p), down_bias (d,), residual x's
    shape. All in x's dtype, bfloat16 or float32; h is rounded to it before its product with down.
    With `keep` it keeps what `feed_forward_backward` takes (bfloat16: 3 bytes a projection, 2 of
    `projected` and 1 of `low`, and 2 a unit); without, as for serving, the projections are never
    in memory."""
    require(x, up, down, up_bias, down_bias, residual)
    is_f32("feed_forward", x, up, down, up_bias, down_bias, residual)
    d, f, p = _kernels("feed_forward", up, down)
    m = rows_of("feed_forward", x, d)
    shaped("feed_forward", "up_bias", up_bias, f, p)
    shaped("feed_forward", "down_bias", down_bias, d)
    shaped("feed_forward", "residual", residual, *x.shape)
    st = ffn.struct(gated=p == 2)
    with on_device(x):
        new = dict(dtype=x.dtype, device=x.device)
        h = torch.empty(*x.shape[:-1], f, **new)
        projected = torch.empty(*x.shape[:-1], f, p, **new) if keep else None
        low = None
        if keep and x.dtype == torch.bfloat16:
            low = torch.empty(*x.shape[:-1], f, p, dtype=torch.int8, device=x.device)
        out = torch.empty(x.shape, **new)
        with span("up + activation"):
            rows_into(x, up, False, m, f * p, d, up_bias, st, None, projected, h, low)
        with span("down"):
            rows_into(h, down, False, m, d, f, down_bias, None, residual, None, out)
    return FeedForward(out, Saved(x, projected, h, low) if keep else None)


def units_backward(dy: torch.Tensor, down: torch.Tensor, projected: torch.Tensor,
                   low: torch.Tensor | None, st: _lib.FfnStruct, m: int, f: int, d: int,
                   sums: bool) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``bux_dense_units_backward`` of tensors already checked: the gradient to `projected`, and with
    `sums` (bfloat16) its low bytes, which its sums over the rows take."""
    dp = torch.empty_like(projected)
    dp_low = None
    if sums and dy.dtype == torch.bfloat16:
        dp_low = torch.empty(dp.shape, dtype=torch.int8, device=dp.device)
    ws, need = room(m, f, d, dy.device)
    if dy.dtype == torch.float32:
        _lib.check(lib().bux_dense_units_backward_f32(
            ptr(dy), ptr(down), m, f, d, ptr(projected), ctypes.byref(st), ptr(dp), ptr(ws), need,
            stream()))
    else:
        _lib.check(lib().bux_dense_units_backward(
            ptr(dy), ptr(down), m, f, d, ptr(projected), ptr(low), ctypes.byref(st), ptr(dp),
            ptr(dp_low), ptr(ws), need, stream()))
    return dp, dp_low


def feed_forward_backward(dy: torch.Tensor, saved: Saved, up: torch.Tensor, down: torch.Tensor,
                          ffn: Ffn = Ffn(), bias: bool = False) -> FeedForwardGrads:
    """Return the gradients of `feed_forward` given dy (x's shape) and what it kept: to x, up
    (d, f, p), down (f, d) and, with `bias`, the biases; `ffn` as the forward's. The residual's
    gradient is dy. Each is rounded to x's dtype from float32 sums; so is d projected before its
    products with up and x, as the MFMAs take it (bfloat16: 2^-8 at most of each term), but not
    before up_bias's sums, which take 24 bits of it."""
    x, projected, h, low = saved
    require(dy, x, projected, h, low, up, down)
    is_f32("feed_forward_backward", x, dy, projected, h, up, down)
    d, f, p = _kernels("feed_forward_backward", up, down)
    m = rows_of("feed_forward_backward", x, d)
    shaped("feed_forward_backward", "dy", dy, *x.shape)
    shaped("feed_forward_backward", "projected", projected, *x.shape[:-1], f, p)
    shaped("feed_forward_backward", "h", h, *x.shape[:-1], f)
    shaped("feed_forward_backward", "low", low, *projected.shape)
    if low is not None and (low.dtype != torch.int8 or low.device != x.device
                            or x.dtype != torch.bfloat16):
        raise ValueError(f"feed_forward_backward: low is int8 beside bfloat16 rows on {x.device}, "
                         f"not {low.dtype} beside {x.dtype} on {low.device}")
    st = ffn.struct(gated=p == 2)
    with on_device(x):
        with span("down dgrad + activation backward"):
            dp, dp_low = units_backward(dy, down, projected, low, st, m, f, d, bias)
        with span("down wgrad"):
            d_down = weight_grad(h, dy)
        dp = dp.view(*x.shape[:-1], f * p)
        with span("up dgrad"):
            dx = torch.empty_like(x)
            rows_into(dp, up, True, m, d, f * p, None, None, None, None, dx)
        with span("up wgrad"):
            d_up = weight_grad(x, dp).view(d, f, p)
        d_up_bias = d_down_bias = None
        if bias:
            with span("bias grads"):
                d_up_bias = slope(dp, m, f * p, sums=True, low=dp_low)[1].view(f, p)
                d_down_bias = slope(dy, m, d, sums=True)[1]
    return FeedForwardGrads(dx, d_up, d_down, d_up_bias, d_down_bias)
