"""The MoE router on MI355X: each token's top-k experts and their weights, from its
logits, in one HIP kernel (``bux_route``).

Mirrors ``MoE._route`` (src/bux/architecture/experts/moe.py:236-273) off training —
no random logits (moe.py:250), no balance or observation taps (moe.py:263-265) — with
``MoE._logits`` (moe.py:275-284) and ``_limit_groups`` (moe.py:474-483). The router's
fields are ``MoEConfig``'s (src/bux/config.py:236-275): ``router``,
``router_logit_scale``, ``normalize_top_k``, ``routed_scaling_factor``,
``num_groups``, ``top_k_groups``; the kernel's columns past the scored experts are the
shared experts' sinks (``shared_expert_sink``, moe.py:143-153).

`route_backward` is its transpose for training (``bux_route_backward``): from the gradients
that the experts' backward gives the picks' weights, and those of losses on the scores and
logits, to the tokens, the router's kernel and its bias.
"""

from typing import NamedTuple

import torch

from bux_amd import _lib
from bux_amd.kernels import lib, on_device, ptr, require, stream, workspace

ROUTERS = {"softmax": _lib.ROUTER_SOFTMAX, "sigmoid": _lib.ROUTER_SIGMOID,
           "sqrtsoftplus": _lib.ROUTER_SQRTSOFTPLUS}


class Routed(NamedTuple):
    """What ``MoE._route`` returns (idx, weights, sinks), and the scores and logits."""

    idx: torch.Tensor  # int32 (t, k): the picks, the largest choice first
    weights: torch.Tensor  # bfloat16 (t, k): their weights
    sinks: torch.Tensor | None  # bfloat16 (t, s): the sinks' weights, None without sinks
    scores: torch.Tensor | None  # float32 (t, scored), if asked for
    logits: torch.Tensor | None  # float32 (t, scored + s), if asked for


def route(x: torch.Tensor, kernel: torch.Tensor, *, top_k: int, scored: int | None = None,
          router: str = "softmax", bias: torch.Tensor | None = None,
          router_logit_scale: float = 1.0, router_bias: torch.Tensor | None = None,
          num_groups: int = 1, top_k_groups: int = 1, normalize_top_k: bool = True,
          routed_scaling_factor: float = 1.0, with_scores: bool = False,
          with_logits: bool = False) -> Routed:
    """Route the bfloat16 tokens `x` (..., d) by the router's bfloat16 `kernel` (d, n):
    the first `scored` (default n) columns score the experts (routed, then zero
    experts), the rest are sinks. `bias` is the router's own float32 bias on the
    logits; `router_bias` the aux-free float32 bias on the choice (the reference's
    ``MoE.router_bias``). Raises ValueError for what the kernel does not take (more
    than 1024 logits, k or top_k_groups over 16, d not a multiple of 16)."""
    require(x, kernel)
    if x.dtype != torch.bfloat16 or kernel.dtype != torch.bfloat16:
        raise TypeError("x and kernel are bfloat16")
    if router not in ROUTERS:
        raise ValueError(f"router {router!r}: one of {sorted(ROUTERS)}")
    lead, d = x.shape[:-1], x.shape[-1]
    if kernel.dim() != 2 or kernel.shape[0] != d:
        raise ValueError(f"kernel {tuple(kernel.shape)} for width {d}")
    n = kernel.shape[1]
    scored = n if scored is None else scored
    xs = x.reshape(-1, d).contiguous()
    t = xs.shape[0]
    dev = x.device
    for name, v, size in (("bias", bias, n), ("router_bias", router_bias, scored)):
        if v is not None and (v.dtype != torch.float32 or v.numel() != size):
            raise ValueError(f"{name}: float32 of {size} elements")
    idx = torch.empty(t, top_k, dtype=torch.int32, device=dev)
    weights = torch.empty(t, top_k, dtype=torch.bfloat16, device=dev)
    sinks = torch.empty(t, n - scored, dtype=torch.bfloat16, device=dev) if n > scored else None
    scores = torch.empty(t, scored, dtype=torch.float32, device=dev) if with_scores else None
    logits = torch.empty(t, n, dtype=torch.float32, device=dev) if with_logits else None
    ws = workspace(lib().bux_route_workspace_size(d, n), dev)
    rc = lib().bux_route(
        ptr(xs), ptr(kernel.contiguous()), ptr(bias), t, d, n, router_logit_scale,
        ROUTERS[router], scored, ptr(router_bias), num_groups, top_k_groups, top_k,
        int(normalize_top_k), routed_scaling_factor, ptr(idx), ptr(weights), ptr(sinks),
        ptr(scores), ptr(logits), ptr(ws), ws.numel(), stream())
    if rc == 1:  # BUX_E_ARGUMENT
        raise ValueError(lib().bux_last_error().decode())
    _lib.check(rc)

    def shaped(v, width):
        return None if v is None else v.reshape(*lead, width)

    return Routed(shaped(idx, top_k), shaped(weights, top_k), shaped(sinks, n - scored),
                  shaped(scores, scored), shaped(logits, n))


class RouteGrads(NamedTuple):
    """What `route_backward` returns."""

    x: torch.Tensor  # bfloat16, x's shape: to the tokens (plus dz)
    kernel: torch.Tensor  # bfloat16 (d, n): to the router's kernel
    bias: torch.Tensor  # float32 (n,): to the router's own bias


def route_backward(x: torch.Tensor, kernel: torch.Tensor, idx: torch.Tensor, logits: torch.Tensor,
                   d_weights: torch.Tensor, *, scored: int | None = None, router: str = "softmax",
                   router_logit_scale: float = 1.0, normalize_top_k: bool = True,
                   routed_scaling_factor: float = 1.0, d_sinks: torch.Tensor | None = None,
                   d_scores: torch.Tensor | None = None, d_logits: torch.Tensor | None = None,
                   dz: torch.Tensor | None = None) -> RouteGrads:
    """The gradients of `route` (of the same x, kernel and settings) given those of its picks'
    weights, `d_weights` (..., k) bfloat16: idx and logits as `route` returned them
    (``with_logits``).

    d_sinks: the sinks' weights' gradient (..., n - scored) bfloat16. d_scores: float32 (...,
    scored), the gradient of a loss on the scores (a balance loss). d_logits: float32 (..., n),
    of one on the logits (a z-loss). dz: bfloat16 of x's shape, the gradient that reached the
    tokens through the experts (`moe.experts_backward`'s "z"), added before x's gradient is
    rounded. The roundings to bfloat16 in the forward pass gradients as they are; the aux-free
    `router_bias` has none. The sums' order is fixed."""
    require(x, kernel, idx, logits, d_weights, d_sinks, d_scores, d_logits, dz)
    if x.dtype != torch.bfloat16 or kernel.dtype != torch.bfloat16:
        raise TypeError("x and kernel are bfloat16")
    if router not in ROUTERS:
        raise ValueError(f"router {router!r}: one of {sorted(ROUTERS)}")
    lead, d = x.shape[:-1], x.shape[-1]
    if kernel.dim() != 2 or kernel.shape[0] != d:
        raise ValueError(f"kernel {tuple(kernel.shape)} for width {d}")
    n = kernel.shape[1]
    scored = n if scored is None else scored
    if not 1 <= scored <= n:
        raise ValueError(f"scored={scored} outside [1, {n}]")
    if idx.dim() != x.dim():
        raise ValueError(f"idx {tuple(idx.shape)} for tokens {tuple(x.shape)}")
    k = idx.shape[-1]
    for name, v, dtype, width in (
            ("idx", idx, torch.int32, k), ("logits", logits, torch.float32, n),
            ("d_weights", d_weights, torch.bfloat16, k),
            ("d_sinks", d_sinks, torch.bfloat16, n - scored),
            ("d_scores", d_scores, torch.float32, scored),
            ("d_logits", d_logits, torch.float32, n), ("dz", dz, torch.bfloat16, d)):
        if v is None:
            continue
        if v.dtype != dtype or v.shape != (*lead, width) or v.device != x.device:
            raise ValueError(f"{name}: {dtype} {(*lead, width)} on {x.device}, not {v.dtype} "
                             f"{tuple(v.shape)} on {v.device}")
    if kernel.device != x.device:
        raise ValueError(f"kernel on {kernel.device} beside tokens on {x.device}")
    t = x.numel() // d if d else 0
    dev = x.device
    with on_device(x):
        # the kernels load 16 bytes at whole 16s
        x, dz = (v if v is None or v.data_ptr() % 16 == 0 else v.clone() for v in (x, dz))
        dx = torch.empty_like(x)
        d_kernel = torch.empty_like(kernel)
        d_bias = torch.empty(n, dtype=torch.float32, device=dev)
        ws = workspace(lib().bux_route_backward_workspace_size(t, d, n), dev)
        rc = lib().bux_route_backward(
            ptr(x), ptr(kernel), t, d, n, router_logit_scale, ROUTERS[router], scored, ptr(idx), k,
            int(normalize_top_k), routed_scaling_factor, ptr(logits), ptr(d_weights), ptr(d_sinks),
            ptr(d_scores), ptr(d_logits), ptr(dz), ptr(dx), ptr(d_kernel), ptr(d_bias), ptr(ws),
            ws.numel(), stream())
    if rc == 1:  # BUX_E_ARGUMENT
        raise ValueError(lib().bux_last_error().decode())
    _lib.check(rc)
    return RouteGrads(dx, d_kernel, d_bias)
