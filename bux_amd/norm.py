"""The tokens' norm before a layer on MI355X, with the residual stream's addition, and its
backward.

The model's ``Norm`` (src/bux/architecture/layers/norm.py:14-78) of rows of any width from 8
to 12288, layernorm or rmsnorm, by `moe.ExpertNorm`'s settings: float32 inside, one rounding
to the rows' type. (`moe.expert_norm_forward`, the norm of the experts' outputs, is tied to
the sort and rounds at every step.) The backward takes the statistics that the forward kept.
"""

import ctypes
from typing import NamedTuple

import torch

from bux_amd import _lib
from bux_amd.kernels import lib, on_device, ptr, require, stream, workspace
from bux_amd.moe import ExpertNorm

MAX_WIDTH = 12288


class Normed(NamedTuple):
    """What `normed` returns."""

    out: torch.Tensor  # the norm of x (+ residual), x's shape and dtype
    summed: torch.Tensor | None  # x + residual in x's dtype, None without a residual
    stats: torch.Tensor | None  # float32 (rows, 2): each row's mean and 1 / rms, if asked for


class NormGrads(NamedTuple):
    """What `normed_backward` returns."""

    x: torch.Tensor  # to x (and to the residual), x's shape and dtype
    scale: torch.Tensor | None  # float32 (d,), None for a norm without a gain
    bias: torch.Tensor | None  # float32 (d,), None for a norm without a bias


def _rows(name: str, x: torch.Tensor, **others: torch.Tensor | None) -> tuple[int, int, bool]:
    """(rows, d, float32) of x (..., d), the others of x's shape and dtype."""
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{name}: bfloat16 or float32 rows, not {x.dtype}")
    if x.dim() < 1 or not 8 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"{name}: rows of 8 to {MAX_WIDTH} columns, not {tuple(x.shape)}")
    for what, t in others.items():
        if t is None:
            continue
        if t.dtype != x.dtype:
            raise TypeError(f"{name}: {what} is {t.dtype} beside {x.dtype} rows")
        if t.shape != x.shape or t.device != x.device:
            raise ValueError(f"{name}: {what} {tuple(t.shape)} on {t.device} beside rows "
                             f"{tuple(x.shape)} on {x.device}")
    d = x.shape[-1]
    return x.numel() // d, d, x.dtype == torch.float32


def _parameter(name: str, what: str, wanted: bool, t: torch.Tensor | None, x: torch.Tensor
               ) -> torch.Tensor | None:
    """The norm's gain or bias: (d,) of x's dtype where the norm has one, else None."""
    if not wanted:
        return None
    if t is None:
        raise ValueError(f"{name}: the norm has a {what}, but none is given")
    if t.dtype != x.dtype:
        raise TypeError(f"{name}: {what} is {t.dtype} beside {x.dtype} rows")
    if t.shape != x.shape[-1:] or t.device != x.device:
        raise ValueError(f"{name}: {what} {tuple(t.shape)} on {t.device} for rows "
                         f"{tuple(x.shape)} on {x.device}")
    return t


def normed(x: torch.Tensor, norm: ExpertNorm = ExpertNorm(), scale: torch.Tensor | None = None,
           bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
           with_stats: bool = True) -> Normed:
    """Norm the rows of x (..., d), bfloat16 or float32. With `residual` (x's shape and dtype)
    it norms their sum, rounded to x's dtype, and returns that sum too (the residual stream
    that goes on). scale and bias are (d,) of x's dtype, where the norm has them. With
    `with_stats` it keeps what `normed_backward` takes."""
    require(x, scale, bias, residual)
    m, d, f32 = _rows("normed", x, residual=residual)
    scale = _parameter("normed", "scale", norm.affine, scale, x)
    bias = _parameter("normed", "bias", norm.bias, bias, x)
    st = norm.struct()
    with on_device(x):
        out = torch.empty_like(x)
        summed = None if residual is None else torch.empty_like(x)
        stats = torch.empty(m, 2, dtype=torch.float32, device=x.device) if with_stats else None
        forward = lib().bux_norm_forward_f32 if f32 else lib().bux_norm_forward
        _lib.check(forward(ptr(x), ptr(residual), m, d, ctypes.byref(st), ptr(scale), ptr(bias),
                           ptr(summed), ptr(out), ptr(stats), stream()))
    return Normed(out, summed, stats)


def normed_backward(dy: torch.Tensor, x: torch.Tensor, stats: torch.Tensor,
                    norm: ExpertNorm = ExpertNorm(), scale: torch.Tensor | None = None,
                    d_summed: torch.Tensor | None = None) -> NormGrads:
    """The gradients of `normed` given dy (x's shape and dtype): to its x (`Normed.summed`
    where a residual was added; then to x and to the residual alike), and to the gain and
    bias, float32 sums over the rows in a fixed order. x is what was normed, stats what the
    forward kept. d_summed (x's shape and dtype): the gradient that reaches the sum past the
    norm, added before the one rounding."""
    require(dy, x, stats, scale, d_summed)
    m, d, f32 = _rows("normed_backward", x, dy=dy, d_summed=d_summed)
    if stats.dtype != torch.float32 or stats.shape != (m, 2) or stats.device != x.device:
        raise ValueError(f"normed_backward: stats are float32 ({m}, 2) on {x.device}, not "
                         f"{stats.dtype} {tuple(stats.shape)} on {stats.device}")
    scale = _parameter("normed_backward", "scale", norm.affine, scale, x)
    dev = x.device
    st = norm.struct()
    with on_device(x):
        dx = torch.empty_like(x)
        d_scale = torch.empty(d, dtype=torch.float32, device=dev) if norm.affine else None
        d_bias = torch.empty(d, dtype=torch.float32, device=dev) if norm.bias else None
        ws = workspace(lib().bux_norm_backward_workspace_size(m, d), dev)
        backward = lib().bux_norm_backward_f32 if f32 else lib().bux_norm_backward
        _lib.check(backward(ptr(dy), ptr(x), ptr(stats), ptr(d_summed), m, d, ctypes.byref(st),
                            ptr(scale), ptr(dx), ptr(d_scale), ptr(d_bias), ptr(ws), ws.numel(),
                            stream()))
    return NormGrads(dx, d_scale, d_bias)
