"""A layer of experts for a few tokens, as a model that is served has them (``csrc/experts.cu``); for many, the same layer is
``grouped.grouped_linear`` twice with ``checkpoints.gated_rows`` in between.

    routes = route_rows(x, router, top)                            # which experts, and with what weights
    y = expert_layer(x, w_up, w_down, routes)                      # y[t] = sum of weight (silu(a) * b) Wd, (a | b) = x[t] Wu

x ``[tokens, width]``, router ``[width, experts]``, w_up ``[experts, width, 2 inner]`` with the gate's columns first, w_down ``[experts,
inner, width]``, y as x: float32, bfloat16 or float16, the same for all operands of a call; x and y possibly with rows further apart than
they are long, the weights any views with contiguous columns. Up to 1,024 experts, 16 choices and, in ``expert_layer``, 128 tokens
and widths of 2^17 (in ``route_rows`` 2^24 and 2^20).
Sums are in float32 and y is rounded once: what passes between the two products keeps 17 bits with bfloat16 weights, 23 with the others. A
product of two float32 is off by 2^-21 of itself at most where both are 2^-112 or more, and by more where they are less: what lies below
2^-136 is lost. A choice that is no expert (negative, as padding has it, or >= the number of experts) gives nothing.

The same call gives the same bits, and a token's result does not depend on what the other tokens are; how many they are fixes the order of
the sums with the other sizes. ``route_rows`` of up to 128 tokens in 16 bits also goes by whether the rows of x and router begin at multiples of
16 bytes: where logits are nearer than float32 sums are exact, a view's choices can be others than its copy's.

Calls run on the current stream of the operands' device and allocate their outputs and scratch from torch's allocator, so they can be
captured, ``expert_layer`` after one call outside a capture (or ``grouped.prepare_device``). Nothing synchronises. A kernel that gives up
waiting raises nothing by itself: ``grouped.check_status``. There is no autograd and no CPU path.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .embedding import _empty, _limits, _scratch
from .grouped import MAX_GROUPS, TYPES, _launch, _matrix, _on_device, _shares_memory, _status_pointer, _weights, _written

MAX_TOP = _lib.MAX_TOP
MAX_TOKENS = _lib.MAX_LAYER_TOKENS
MAX_ROUTED = 1 << 24                          # tokens of route_rows


class Routes(NamedTuple):
    """``experts``: int32 ``[tokens, top]``; ``weights``: float32 ``[tokens, top]``."""
    experts: torch.Tensor
    weights: torch.Tensor


def _kind(what: str, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor) -> int:
    dtype = x.dtype
    kind = TYPES.get(dtype)
    if kind is None or a.dtype != dtype or b.dtype != dtype:
        raise ValueError(f"{what}: the operands must have the same type, float32, bfloat16 or float16")
    return kind


def route_rows(x: torch.Tensor, router: torch.Tensor, top: int, normalise: bool = True) -> Routes:
    """The ``top`` experts with the largest logits ``x router`` of each token, in falling order, equal ones by number (NaN is chosen last),
    and their weights: the softmax over the chosen logits, or over all (``normalise=False``). Up to 2^24 tokens."""
    what = "route_rows"
    tokens, width, stride = _matrix(what, "x", x)
    _, count, router_stride = _matrix(what, "router", router, rows=width)
    kind = _kind(what, x, router, router)
    _limits(what, tokens, width, MAX_ROUTED)
    if count > MAX_GROUPS:
        raise ValueError(f"{what}: more than {MAX_GROUPS} experts")
    top = int(top)
    if not 1 <= top <= MAX_TOP or top > count:
        raise ValueError(f"{what}: 1 to {min(MAX_TOP, count)} choices")
    index, device = _on_device(what, x, router), x.device
    routes = Routes(_empty(tokens, top, torch.int32, device), _empty(tokens, top, torch.float32, device))
    if tokens:
        a = _lib.RouteStruct(kind, tokens, width, count, top, bool(normalise), x.data_ptr(), router.data_ptr(),
                             routes.experts.data_ptr(), routes.weights.data_ptr(), stride, router_stride)
        _lib.check(_launch(index, _lib.load().fmb_route_rows, ctypes.byref(a)), "fmb_route_rows")
    return routes


def expert_layer(x: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, routes: Routes, out: torch.Tensor | None = None) -> torch.Tensor:
    """``y[t] = sum over j of weights[t, j] (silu(a) * b) w_down[e]``, ``(a | b) = x[t] w_up[e]``, ``e = experts[t, j]``."""
    what = "expert_layer"
    tokens, width, stride = _matrix(what, "x", x)
    kind = _kind(what, x, w_up, w_down)
    count, up_k, up_n, up_group, up_row = _weights(what, "w_up", w_up)
    down_count, inner, down_n, down_group, down_row = _weights(what, "w_down", w_down)
    if not 1 <= count <= MAX_GROUPS or down_count != count or up_k != width or down_n != width or inner < 1 or up_n != 2 * inner:
        raise ValueError(f"{what}: w_up {tuple(w_up.shape)} and w_down {tuple(w_down.shape)} must be [experts, {width}, 2 inner] and "
                         f"[experts, inner, {width}] of 1 to {MAX_GROUPS} experts")
    chosen, weights = routes
    if tokens > MAX_TOKENS:
        raise ValueError(f"{what}: {tokens} tokens, of {MAX_TOKENS} at most: grouped_linear is for more")
    shape = chosen.shape
    if chosen.dtype != torch.int32 or weights.dtype != torch.float32 or len(shape) != 2 or shape != weights.shape or \
            shape[0] != tokens or not 1 <= shape[1] <= MAX_TOP or not chosen.is_contiguous() or not weights.is_contiguous():
        raise ValueError(f"{what}: routes must be as route_rows returns them, for {tokens} tokens and 1 to {MAX_TOP} choices")
    index = _on_device(what, x, w_up, w_down, chosen, weights)
    given = out is not None
    if given:
        out_stride = _matrix(what, "out", out, width, tokens)[2]
        if out.dtype != x.dtype:
            raise ValueError(f"{what}: out must have the input's type")
        _on_device(what, x, out)
        if any(_shares_memory(out, t) for t in (x, w_up, w_down, chosen, weights)):
            raise ValueError(f"{what}: out shares memory with an operand")
    else:
        out, out_stride = _empty(tokens, width, x.dtype, x.device), width
    if tokens:
        lib = _lib.load()
        a = _lib.ExpertsStruct(kind, tokens, count, shape[1], width, inner, x.data_ptr(), w_up.data_ptr(), w_down.data_ptr(),
                               chosen.data_ptr(), weights.data_ptr(), out.data_ptr(), stride, out_stride, up_group, up_row, down_group,
                               down_row, None, _status_pointer(index))
        call = ctypes.byref(a)
        scratch = _scratch(lib.fmb_expert_layer_scratch(call), torch.float32, x.device)
        a.scratch = scratch.data_ptr()
        _lib.check(_launch(index, lib.fmb_expert_layer, call), "fmb_expert_layer")
        if given:
            _written(out)
    return out


__all__ = ["Routes", "route_rows", "expert_layer", "MAX_TOP", "MAX_TOKENS"]
