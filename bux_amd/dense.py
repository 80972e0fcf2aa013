"""A dense matrix product on MI355X with its bias, activation and residual in the epilogue, and
its backward: the projections around a layer's experts.

float32 sums with one rounding of each output, bfloat16 or float32 throughout; in the backward
with an activation the gradient before the products is rounded too. `mlp` makes the
dense feed-forward block of them; the experts' own products are `grouped`, `grouped_mxfp8` and
`grouped_int8`.
"""

import ctypes
from typing import NamedTuple

import torch

from bux_amd import _lib
from bux_amd.kernels import lib, on_device, ptr, require, stream, workspace
from bux_amd.moe import Ffn


class Product(NamedTuple):
    """What `product` returns."""

    out: torch.Tensor  # (..., n), x's dtype
    product: torch.Tensor | None  # x w + bias before the activation, if asked for


class ProductGrads(NamedTuple):
    """What `product_backward` returns. (The residual's gradient is dy.)"""

    x: torch.Tensor  # x's shape
    w: torch.Tensor  # w's shape
    bias: torch.Tensor | None  # (n,), None if not asked for


def is_f32(name: str, x: torch.Tensor, *others: torch.Tensor | None) -> bool:
    """Whether the op runs in float32: every tensor given has x's dtype and lies on its GPU."""
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{name}: bfloat16 or float32, not {x.dtype}")
    for t in others:
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"{name}: a {t.dtype} tensor beside {x.dtype} rows")
        if t is not None and t.device != x.device:
            raise ValueError(f"{name}: a tensor on {t.device} beside rows on {x.device}")
    return x.dtype == torch.float32


def shaped(name: str, what: str, t: torch.Tensor | None, *shape: int) -> None:
    """Raise unless t, where given, has this shape."""
    if t is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name}: {what} is {shape}, not {tuple(t.shape)}")


def rows_of(name: str, x: torch.Tensor, width: int) -> int:
    """The rows of x (..., width)."""
    if x.dim() < 1 or x.shape[-1] != width or width < 1:
        raise ValueError(f"{name}: rows of {width}, not {tuple(x.shape)}")
    return x.numel() // width


def _sides(name: str, w: torch.Tensor, transposed: bool) -> tuple[int, int]:
    if w.dim() != 2 or w.numel() == 0:
        raise ValueError(f"{name}: a kernel (k, n), not {tuple(w.shape)}")
    return (w.shape[1], w.shape[0]) if transposed else (w.shape[0], w.shape[1])


def _plain(activation: str | None) -> _lib.FfnStruct | None:
    return None if activation is None else Ffn(activation).struct(gated=False)


def _ref(st: _lib.FfnStruct | None):
    return None if st is None else ctypes.byref(st)


def room(m: int, n: int, k: int, dev: torch.device) -> tuple[torch.Tensor | None, int]:
    """The workspace of a product of m rows, n columns and k contracted, and its bytes."""
    need = lib().bux_dense_workspace_size(m, n, k)
    return (workspace(need, dev), need) if need else (None, 0)


def rows_into(x: torch.Tensor, w: torch.Tensor, transposed: bool, m: int, n: int, k: int,
              bias: torch.Tensor | None, st: _lib.FfnStruct | None,
              residual: torch.Tensor | None, product: torch.Tensor | None, out: torch.Tensor,
              low: torch.Tensor | None = None) -> None:
    """``bux_dense_rows`` of tensors already checked."""
    ws, need = room(m, n, k, x.device)
    if x.dtype == torch.float32:
        _lib.check(lib().bux_dense_rows_f32(
            ptr(x), ptr(w), int(transposed), m, n, k, ptr(bias), _ref(st), ptr(residual),
            ptr(product), ptr(out), ptr(ws), need, stream()))
    else:
        _lib.check(lib().bux_dense_rows(
            ptr(x), ptr(w), int(transposed), m, n, k, ptr(bias), _ref(st), ptr(residual),
            ptr(product), ptr(low), ptr(out), ptr(ws), need, stream()))


def product(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None,
            activation: str | None = None, residual: torch.Tensor | None = None,
            transposed: bool = False, with_product: bool = False) -> Product:
    """Return ``act(x w + bias) + residual`` of the rows x (..., k) and the kernel w (k, n), or
    with `transposed` (n, k): bias (n,), residual (..., n), activation one of
    ``_lib.ACTIVATIONS`` or None. With `with_product` it keeps ``x w + bias``, which
    `product_backward` takes where there is an activation. All in x's dtype, bfloat16 or
    float32."""
    require(x, w, bias, residual)
    is_f32("product", x, w, bias, residual)
    k, n = _sides("product", w, transposed)
    m = rows_of("product", x, k)
    shape = (*x.shape[:-1], n)
    shaped("product", "bias", bias, n)
    shaped("product", "residual", residual, *shape)
    st = _plain(activation)
    with on_device(x):
        out = torch.empty(shape, dtype=x.dtype, device=x.device)
        kept = torch.empty(shape, dtype=x.dtype, device=x.device) if with_product else None
        rows_into(x, w, transposed, m, n, k, bias, st, residual, kept, out)
    return Product(out, kept)


def weight_grad(x: torch.Tensor, dy: torch.Tensor) -> torch.Tensor:
    """Return ``x^T dy`` (k, n) of the rows x (..., k) and dy (..., n), in their dtype; 0 for no
    rows."""
    require(x, dy)
    f32 = is_f32("weight_grad", x, dy)
    if x.dim() < 1 or dy.dim() < 1:
        raise ValueError("weight_grad: rows, not a scalar")
    k, n = x.shape[-1], dy.shape[-1]
    m = rows_of("weight_grad", x, k)
    if dy.shape[:-1] != x.shape[:-1] or n < 1:
        raise ValueError(f"weight_grad: rows {tuple(x.shape)} and {tuple(dy.shape)}")
    with on_device(x):
        dw = torch.empty(k, n, dtype=x.dtype, device=x.device)
        ws, need = room(k, n, m, x.device)
        contract = lib().bux_dense_contract_f32 if f32 else lib().bux_dense_contract
        _lib.check(contract(ptr(x), ptr(dy), m, k, n, ptr(dw), ptr(ws), need, stream()))
    return dw


def slope(dy: torch.Tensor, m: int, n: int, product: torch.Tensor | None = None,
          st: _lib.FfnStruct | None = None, sums: bool = False, low: torch.Tensor | None = None
          ) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """``bux_dense_slope`` of dy (m, n) (its sums with its low bytes, `low`), already checked: dy
    times the activation's derivative at `product` (None without one), and with `sums` that
    gradient's sums over the rows."""
    dz = torch.empty_like(dy) if product is not None else None
    out = torch.empty(n, dtype=dy.dtype, device=dy.device) if sums else None
    if dz is None and out is None:
        return None, None
    need = lib().bux_dense_slope_workspace_size(m, n) if sums else 0
    ws = workspace(need, dy.device) if need else None
    if dy.dtype == torch.float32:
        _lib.check(lib().bux_dense_slope_f32(ptr(dy), ptr(product), _ref(st), m, n, ptr(dz),
                                             ptr(out), ptr(ws), need, stream()))
    else:
        _lib.check(lib().bux_dense_slope(ptr(dy), ptr(low), ptr(product), _ref(st), m, n, ptr(dz),
                                         ptr(out), ptr(ws), need, stream()))
    return dz, out


def product_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor,
                     activation: str | None = None, product: torch.Tensor | None = None,
                     transposed: bool = False, bias: bool = False) -> ProductGrads:
    """Return the gradients of `product` to x, w and, with `bias`, its bias, given dy (..., n):
    with an activation, `product` is what the forward kept. The residual's gradient is dy. Each
    is rounded to x's dtype from float32 sums. With an activation in bfloat16, dz = dy act'(product)
    is rounded to bfloat16 too before its products with w and x, as the MFMAs take it (a bfloat16
    step of 2^-8 at most in each term), not before the bias's sums; and act' is taken at the kept
    `product`, itself rounded."""
    require(dy, x, w, product)
    is_f32("product_backward", x, dy, w, product)
    k, n = _sides("product_backward", w, transposed)
    m = rows_of("product_backward", x, k)
    shaped("product_backward", "dy", dy, *x.shape[:-1], n)
    if (activation is None) != (product is None):
        raise ValueError("product_backward: an activation's gradient takes the kept product, and "
                         "only that")
    shaped("product_backward", "product", product, *dy.shape)
    st = _plain(activation)
    with on_device(x):
        dz, d_bias = slope(dy, m, n, product, st, bias)
        dz = dy if dz is None else dz
        dx = torch.empty_like(x)
        rows_into(dz, w, not transposed, m, k, n, None, None, None, None, dx)
        dw = weight_grad(dz, x) if transposed else weight_grad(x, dz)
    return ProductGrads(dx, dw, d_bias)
