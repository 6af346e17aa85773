"""What a backward pass needs of a forward one, kept in 8 bits (``csrc/checkpoints.cu``): rows as e4m3 codes in units of a power of two
per 32 columns, the gate of an expert's two matrices, and the backward pass from them.

    held = hold_rows(x)                                            # of a grouped linear: 1.03 bytes a value
    h, held_u = gated_rows(u, hold=True)                           # u = (a | b), h = silu(a) * b, u held on the way
    ...
    du, h = gated_rows_gradient(held_u, dh)                        # h anew, so that it need not be kept
    dw = held_weight_gradient(held, dy, groups)                    # dW[g] = sum over its rows of x[r]^T dy[r], fp32

A block's unit is the smallest power of two with |x| <= 448 units, so a value is off by at most 2^-4 of itself, or by half of the smallest
code (2^-10 units) where it is far below its block's largest. Read back, a held value is a number of its own type with no further rounding:
the products with it are those of ``grouped_linear_weight_gradient`` with ``release_rows(held)`` (the same bits where k is a multiple of 8).
Units are between 2^-117 and 2^120, in float16 2^-15 and 2^8; in the highest, codes end at 240. What is not finite is held as NaN, and leaves
the others of its block as they are.

Rows: float32, bfloat16 or float16, up to 2^30 of up to 2^20 columns, possibly further apart than they are long. Gates are computed in
float32 and rounded once. Calls run on the current stream of the operands' device and allocate their outputs and scratch from torch's
allocator, so they can be captured (``held_weight_gradient`` after one call of its kind outside a capture). Nothing synchronises. There is no
autograd and no CPU path.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .embedding import _empty, _limits
from .grouped import TYPES, RowGroups, _launch, _matrix, _on_device, _shares_memory, _weight_gradient, _written

BLOCK = _lib.HELD_BLOCK


class HeldRows(NamedTuple):
    """``codes``: float8_e4m3fn ``[rows, columns]``; ``exponents``: uint8 ``[rows, parts * ceil(columns / parts / 32)]``, of each block's
    unit, plus 127; ``dtype``: the rows' type. With 2 ``parts`` each half of the columns has blocks of its own."""
    codes: torch.Tensor
    exponents: torch.Tensor
    dtype: torch.dtype
    parts: int = 1


def _blocks(columns: int, parts: int) -> int:
    return parts * -(-(columns // parts) // BLOCK)


def _kind(what: str, dtype: torch.dtype) -> int:
    if dtype not in TYPES:
        raise ValueError(f"{what}: rows must be float32, bfloat16 or float16")
    return TYPES[dtype]


def _parts(what: str, columns: int, parts: int) -> None:
    if parts not in (1, 2) or columns % parts:
        raise ValueError(f"{what}: 1 or 2 parts of the same size")


def _held(what: str, held: HeldRows, parts: int | None = None):
    """(rows, columns) of held rows, checked."""
    codes, exponents = held.codes, held.exponents
    _kind(what, held.dtype)
    if codes.dim() != 2 or codes.dtype != torch.float8_e4m3fn or not codes.is_contiguous() or exponents.dtype != torch.uint8 or \
            not exponents.is_contiguous() or codes.shape[1] < 1:
        raise ValueError(f"{what}: held rows must be as hold_rows returns them")
    rows, columns = codes.shape
    _limits(what, rows, columns)
    _parts(what, columns, held.parts)
    if parts is not None and held.parts != parts:
        raise ValueError(f"{what}: rows held in {parts} part{'s' if parts > 1 else ''} are expected, these have {held.parts}")
    if tuple(exponents.shape) != (rows, _blocks(columns, held.parts)):
        raise ValueError(f"{what}: exponents must be {(rows, _blocks(columns, held.parts))}, got {tuple(exponents.shape)}")
    return rows, columns


def _new_held(rows: int, columns: int, parts: int, like: torch.Tensor) -> HeldRows:
    device = like.device
    return HeldRows(_empty(rows, columns, torch.float8_e4m3fn, device), _empty(rows, _blocks(columns, parts), torch.uint8, device), like.dtype, parts)


def _struct(kind: int, rows: int, columns: int, parts: int, held: HeldRows | None, x=(None, 0), h=(None, 0), dh=(None, 0), du=(None, 0)):
    """The C call's arguments; x, h, dh, du as (tensor, row stride)."""
    at = [t if t is None else t.data_ptr() for t, _ in (x, h, dh, du)]
    codes, exponents = (None, None) if held is None else (held[0].data_ptr(), held[1].data_ptr())
    return _lib.HeldStruct(kind, rows, columns, parts, at[0], codes, exponents, *at[1:], x[1], h[1], dh[1], du[1])


def _given(what: str, name: str, out: torch.Tensor | None, rows: int, columns: int, like: torch.Tensor, dtype: torch.dtype, *operands):
    """(output, row stride): one that is given, checked, or a new one."""
    if out is None:
        return _empty(rows, columns, dtype, like.device), columns
    stride = _matrix(what, name, out, columns, rows)[2]
    if out.dtype != dtype:
        raise ValueError(f"{what}: {name} must be {dtype}")
    _on_device(what, like, out)
    if any(_shares_memory(out, t) for t in operands):
        raise ValueError(f"{what}: {name} shares memory with an operand")
    return out, stride


def hold_rows(x: torch.Tensor, parts: int = 1) -> HeldRows:
    """The rows x ``[rows, columns]`` in 8 bits."""
    what = "hold_rows"
    rows, columns, stride = _matrix(what, "x", x)
    kind = _kind(what, x.dtype)
    _limits(what, rows, columns)
    _parts(what, columns, parts)
    index = _on_device(what, x)
    held = _new_held(rows, columns, parts, x)
    if rows:
        a = _struct(kind, rows, columns, parts, held, x=(x, stride))
        _lib.check(_launch(index, _lib.load().fmb_hold_rows, ctypes.byref(a)), "fmb_hold_rows")
    return held


def release_rows(held: HeldRows, out: torch.Tensor | None = None) -> torch.Tensor:
    """The rows that are held, ``[rows, columns]`` in their own type."""
    what = "release_rows"
    rows, columns = _held(what, held)
    index = _on_device(what, held.codes, held.exponents)
    x, stride = _given(what, "out", out, rows, columns, held.codes, held.dtype, held.codes, held.exponents)
    if rows:
        a = _struct(TYPES[held.dtype], rows, columns, held.parts, held, h=(x, stride))
        _lib.check(_launch(index, _lib.load().fmb_release_rows, ctypes.byref(a)), "fmb_release_rows")
        if out is not None:
            _written(out)
    return x


def gated_rows(u: torch.Tensor, hold: bool = False, out: torch.Tensor | None = None):
    """``h = silu(a) * b`` for rows u = (a | b): u ``[rows, 2 f]``, h ``[rows, f]`` of the same type. ``hold=True`` returns (h, u held in two
    parts)."""
    what = "gated_rows"
    rows, columns, stride = _matrix(what, "u", u)
    kind = _kind(what, u.dtype)
    _limits(what, rows, columns)
    _parts(what, columns, 2)
    index = _on_device(what, u)
    h, h_stride = _given(what, "out", out, rows, columns // 2, u, u.dtype, u)
    held = _new_held(rows, columns, 2, u) if hold else None
    if rows:
        a = _struct(kind, rows, columns, 2, held, x=(u, stride), h=(h, h_stride))
        _lib.check(_launch(index, _lib.load().fmb_gated_rows, ctypes.byref(a)), "fmb_gated_rows")
        if out is not None:
            _written(out)
    return (h, held) if hold else h


def gated_rows_gradient(u: HeldRows | torch.Tensor, dh: torch.Tensor, out: torch.Tensor | None = None, recompute: bool = True):
    """(du, h) of ``h = silu(a) * b`` from dh ``[rows, f]``: ``du = (dh b s (1 + a (1 - s)) | dh a s)`` with s = 1 / (1 + exp(-a)). u = (a | b)
    as ``gated_rows`` has held it, or the rows themselves. h is computed anew with it, for the gradient of the weights behind the gate;
    ``recompute=False`` returns (du, None). ``out``: where du goes."""
    what = "gated_rows_gradient"
    if isinstance(u, HeldRows):
        rows, columns = _held(what, u, 2)
        operands, dtype, source = (u.codes, u.exponents), u.dtype, {}
    else:
        rows, columns, stride = _matrix(what, "u", u)
        _kind(what, u.dtype)
        _limits(what, rows, columns)
        _parts(what, columns, 2)
        operands, dtype, source = (u,), u.dtype, {"x": (u, stride)}
    dh_stride = _matrix(what, "dh", dh, columns // 2, rows)[2]
    if dh.dtype != dtype:
        raise ValueError(f"{what}: dh must have the rows' type, {dtype}")
    index = _on_device(what, dh, *operands)
    du, du_stride = _given(what, "out", out, rows, columns, dh, dtype, dh, *operands)
    h = _empty(rows, columns // 2, dtype, dh.device) if recompute else None
    if rows:
        a = _struct(TYPES[dtype], rows, columns, 2, None if source else u, dh=(dh, dh_stride), du=(du, du_stride),
                    h=(h, columns // 2), **source)
        _lib.check(_launch(index, _lib.load().fmb_gated_rows_gradient, ctypes.byref(a)), "fmb_gated_rows_gradient")
        if out is not None:
            _written(out)
    return du, h


def held_weight_gradient(held: HeldRows, dy: torch.Tensor, groups: RowGroups, out: torch.Tensor | None = None,
                         accumulate: bool = False) -> torch.Tensor:
    """``grouped.grouped_linear_weight_gradient`` with x as ``hold_rows`` has kept it: float32 ``[groups, k, n]``."""
    what = "held_weight_gradient"
    rows, columns = _held(what, held, 1)
    _on_device(what, held.codes, held.exponents)
    return _weight_gradient(what, held.codes, columns, held.dtype, dy, groups, out, accumulate, held.exponents)


__all__ = ["HeldRows", "hold_rows", "release_rows", "gated_rows", "gated_rows_gradient", "held_weight_gradient", "BLOCK"]
