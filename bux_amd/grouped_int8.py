"""The experts' products in 8-bit integers on MI355X, for serving: rows of tokens quantized with
a scale a row, the experts' kernels with a scale an output column, exact 32-bit integer sums.

It stands beside the MXFP8 products (`grouped_mxfp8`) and takes the same sort, group sizes and
tile lists; `moe.in_int8` and `moe.experts_int8` run the routed experts with it.
"""

from typing import NamedTuple

import torch

from bux_amd import _lib
from bux_amd.grouped_mxfp8 import K_ALIGN, TileList, tiles_of, whole
from bux_amd.kernels import lib, on_device, ptr, require, stream, workspace

MAX_K = 131072  # 127^2 K stays within 32 bits


class Int8(NamedTuple):
    """Rows in 8-bit integers in the GEMM's tiled layout: row r's code k at [k // 64, r, k % 64],
    K padded with zeros to whole 128s; a stack of matrices has a leading axis."""

    values: torch.Tensor  # int8 (..., K / 64, rows, 64)
    scales: torch.Tensor  # float32 (..., rows): a row's value is its codes times its scale


def _f32(name: str, x: torch.Tensor) -> bool:
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{name}: bfloat16 or float32 values, not {x.dtype}")
    return x.dtype == torch.float32


def quantized(x: torch.Tensor, filled: torch.Tensor | None = None,
              index: torch.Tensor | None = None, index_div: int = 1,
              height: int | None = None) -> Int8:
    """Return the rows of x (r, c), bfloat16 or float32, in 8-bit integers: the nearest to ``127
    x / max |x|`` of the row (the even one at a tie), the row's scale ``max |x| / 127``. With
    `index` (int32) the rows are ``x[index // index_div]`` (a row of 0 where that lies outside
    x), `height` (at least the rows, and by default those) rows in the copy: those past the
    rows, or from `filled` (an int32 on the device) on, are 0. A row that holds an infinity or a
    NaN has that as its scale and codes of 0."""
    require(x, filled, index)
    f32 = _f32("quantized", x)
    if x.dim() != 2 or not 1 <= x.shape[1] <= MAX_K:
        raise ValueError(f"quantized: a matrix of 1 to {MAX_K} columns, not {tuple(x.shape)}")
    for name, t in (("index", index), ("filled", filled)):
        if t is not None and (t.dtype != torch.int32 or t.device != x.device):
            raise ValueError(f"quantized: {name} is int32 on {x.device}, not {t.dtype} on {t.device}")
    if index_div < 1:
        raise ValueError(f"quantized: index_div={index_div}")
    sources, cols = x.shape
    rows = sources if index is None else index.numel()
    height = rows if height is None else height
    if height < rows:
        raise ValueError(f"quantized: height={height} for {rows} rows")
    with on_device(x):
        out = Int8(torch.empty(whole(cols, K_ALIGN) // 64, height, 64, dtype=torch.int8,
                               device=x.device),
                   torch.empty(height, dtype=torch.float32, device=x.device))
        quantize = lib().bux_int8_quantize_f32 if f32 else lib().bux_int8_quantize
        need = 0 if index is None else lib().bux_int8_quantize_workspace_size(sources, rows, cols)
        ws = workspace(need, x.device) if need else None
        _lib.check(quantize(ptr(x), ptr(index), index_div, sources, rows, cols, height, ptr(filled),
                            ptr(out.values), ptr(out.scales), ptr(ws), need, stream()))
    return out


def quantized_kernels(w: torch.Tensor) -> Int8:
    """Return the kernels w (g, k, n), bfloat16 or float32, in 8-bit integers as `rows` takes
    them: each column along k with a scale of its own, as n rows of K codes a group. Once, as
    the weights are loaded."""
    require(w)
    f32 = _f32("quantized_kernels", w)
    if w.dim() != 3 or not 1 <= w.shape[1] <= MAX_K or w.shape[2] < 1:
        raise ValueError(f"quantized_kernels: (g, k, n) of k up to {MAX_K}, not {tuple(w.shape)}")
    g, k, n = w.shape
    with on_device(w):
        out = Int8(torch.empty(g, whole(k, K_ALIGN) // 64, n, 64, dtype=torch.int8, device=w.device),
                   torch.empty(g, n, dtype=torch.float32, device=w.device))
        quantize = (lib().bux_int8_quantize_columns_f32 if f32 else lib().bux_int8_quantize_columns)
        _lib.check(quantize(ptr(w), g, k, n, ptr(out.values), ptr(out.scales), stream()))
    return out


def rows(a: Int8, b: Int8, sizes: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
         height: int | None = None, tiles: TileList | None = None,
         bias: torch.Tensor | None = None) -> torch.Tensor:
    """Return each group's rows of a times its kernel of b, (height, n) in `dtype` (bfloat16 or
    float32): the integer sums times the row's and the column's scale, plus the group's row of
    `bias` (g, n), rounded once; rows past the groups are 0. sizes: int32 (g,), each group's
    rows of a, one group's after another's. height: y's rows, by default a's. tiles:
    ``grouped_mxfp8.tiles_of(sizes, a's rows, height)``, made here if None. n a multiple of 4."""
    require(a.values, a.scales, b.values, b.scales, sizes, bias)
    if dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"rows: a bfloat16 or float32 product, not {dtype}")
    if a.values.dim() != 3 or b.values.dim() != 4 or a.values.shape[0] != b.values.shape[1]:
        raise ValueError(f"rows: codes {tuple(a.values.shape)} times {tuple(b.values.shape)}")
    groups, chunks, n, _ = b.values.shape
    m = a.values.shape[1]
    for t, shape, kind in ((a.values, (chunks, m, 64), torch.int8), (a.scales, (m,), torch.float32),
                           (b.values, (groups, chunks, n, 64), torch.int8),
                           (b.scales, (groups, n), torch.float32),
                           (sizes, (groups,), torch.int32), (bias, (groups, n), dtype)):
        if t is not None and (t.shape != shape or t.dtype != kind or t.device != a.values.device):
            raise ValueError(f"rows: {kind} {shape} on {a.values.device}, not {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")
    if n % 4 != 0:
        raise ValueError(f"rows: n={n} is not a multiple of 4")
    height = m if height is None else height
    with on_device(a.values):
        if tiles is None:
            tiles = tiles_of(sizes, m, height)
        elif (tiles.groups, tiles.m, tiles.height) != (groups, m, height):
            raise ValueError(f"rows: a tile list for {tiles.groups} groups, m={tiles.m}, "
                             f"height={tiles.height}, not {groups}, {m}, {height}")
        y = torch.empty(height, n, dtype=dtype, device=a.values.device)
        _lib.check(lib().bux_int8_grouped_rows_listed(
            ptr(a.values), ptr(a.scales), ptr(b.values), ptr(b.scales), ptr(tiles.buffer),
            tiles.buffer.numel(), groups, m, n, 64 * chunks, height,
            _lib.BF16 if dtype == torch.bfloat16 else _lib.F32, ptr(bias), ptr(y), stream()))
    return y
