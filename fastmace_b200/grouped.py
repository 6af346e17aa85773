"""Products with one matrix per group of rows -- the species-dependent linear of an interaction (``l{t}.skip.{l}``), or the
experts of a layer -- with any number of rows per group, and their gradients (``csrc/grouping.cu``, ``csrc/grouped.cu``).

    groups = group_rows(species, n_species)                         # rows by group, once per set of atoms
    y  = grouped_linear(x, weight, groups)                          # y[r]  = x[r] W[g(r)]
    dx = grouped_linear_input_gradient(dy, weight, groups)          # dx[r] = dy[r] W[g(r)]^T
    dw = grouped_linear_weight_gradient(x, dy, groups)              # dW[g] = sum over its rows of x[r]^T dy[r], fp32

Rows keep their places: row r of ``y`` belongs to row r of ``x`` whatever the order of the groups. ``x`` and ``dy`` may be
views whose rows are further apart than they are long (a component of ``[atom][component][channel]`` features), ``weight``
any ``[groups, k, n]`` view with contiguous columns (``w["l1.skip.0"].permute(1, 0, 2)``). Types: float32, bfloat16, float16,
the same for all operands of a call; sums are in float32 at least (float32 operands keep their 24 bits), the weight gradient
is float32 whatever the operands'. A row of no group (key negative or >= the number of groups) is zero in an output the call
allocates, left as it was in one that is given, and takes no part in a weight gradient.

Calls run on the current stream of the operands' device and allocate their outputs and scratch from torch's allocator, so
they can be captured. There is no autograd and no CPU path.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib

MAX_GROUPS = _lib.MAX_GROUPS
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class RowGroups(NamedTuple):
    """``rows``: int32, the row numbers of group 0, then of group 1, ..., then of the rows without a group; ``offsets``:
    int32 ``[groups + 1]``, where each group starts."""
    rows: torch.Tensor
    offsets: torch.Tensor


_status: dict[torch.device, torch.Tensor] = {}


def _status_of(device: torch.device) -> torch.Tensor:
    if device not in _status:
        if torch.cuda.is_current_stream_capturing():
            raise _lib.Fmb200Error("call grouped.prepare_device() before capturing the first grouped product")
        _status[device] = torch.zeros((), dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()       # other streams may use it from here on
    return _status[device]


def prepare_device(device="cuda") -> None:
    """Makes the device's status word; needed only where the first call on a device would be a captured one."""
    device = torch.device(device)
    _status_of(device if device.index is not None else torch.device("cuda", torch.cuda.current_device()))


def check_status(device="cuda") -> None:
    """Raises if a grouped product on ``device`` gave up waiting since the last check (synchronises)."""
    device = torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    word = _status.get(device)
    if word is not None and int(word.item()) & _lib.STATUS_TENSOR_TIMEOUT:
        word.zero_()
        raise _lib.Fmb200Error("a tensor-core kernel gave up waiting (FMB_STATUS_TENSOR_TIMEOUT)")


def _on_device(what: str, *tensors: torch.Tensor) -> torch.device:
    device = tensors[0].device
    for t in tensors:
        if not t.is_cuda:
            raise ValueError(f"{what}: the operands must be CUDA tensors, there is no CPU path")
        if t.device != device:
            raise ValueError(f"{what}: the operands are on different devices")
    return device


def group_rows(keys: torch.Tensor, n_groups: int) -> RowGroups:
    """Rows by group for ``keys`` (int32 or int64, one per row): a stable order, so equal keys keep the order of their rows.
    1 to 1,024 groups. Does not synchronise."""
    if keys.dim() != 1 or keys.dtype not in (torch.int32, torch.int64):
        raise ValueError("group_rows: keys must be one int32 or int64 per row")
    if not 1 <= int(n_groups) <= MAX_GROUPS:
        raise ValueError(f"group_rows: 1 to {MAX_GROUPS} groups")
    device = _on_device("group_rows", keys)
    if keys.shape[0] > 1 and keys.stride(0) != 1:
        keys = keys.contiguous()
    rows = keys.shape[0]
    lib = _lib.load()
    with torch.cuda.device(device):
        out = RowGroups(torch.empty(rows, dtype=torch.int32, device=device),
                        torch.empty(int(n_groups) + 1, dtype=torch.int32, device=device))
        need = lib.fmb_group_rows_scratch(rows, int(n_groups))
        scratch = torch.empty(need, dtype=torch.int32, device=device) if need else None
        _lib.check(lib.fmb_group_rows(keys.data_ptr(), keys.element_size(), rows, int(n_groups), out.rows.data_ptr(),
                                      out.offsets.data_ptr(), scratch.data_ptr() if need else None, _lib.current_stream()),
                   "fmb_group_rows")
    return out


def _matrix(what: str, name: str, t: torch.Tensor, shape: tuple | None = None) -> torch.Tensor:
    if t.dim() != 2 or (shape is not None and tuple(t.shape) != shape):
        raise ValueError(f"{what}: {name} must be {shape if shape else 'a matrix'}, got {tuple(t.shape)}")
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{what}: {name} must have contiguous rows that do not overlap")
    return t


def _weights(what: str, name: str, t: torch.Tensor) -> torch.Tensor:
    if t.dim() != 3:
        raise ValueError(f"{what}: {name} must be [groups, k, n], got {tuple(t.shape)}")
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise ValueError(f"{what}: the columns of {name} must be contiguous")
    return t


def _groups(what: str, groups: RowGroups, rows: int, n_groups: int | None) -> int:
    order, offsets = groups
    for t in (order, offsets):
        if t.dim() != 1 or t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError(f"{what}: groups must be as group_rows returns them")
    if order.shape[0] != rows:
        raise ValueError(f"{what}: groups of {order.shape[0]} rows for {rows} rows")
    count = offsets.shape[0] - 1
    if not 1 <= count <= MAX_GROUPS:
        raise ValueError(f"{what}: 1 to {MAX_GROUPS} groups")
    if n_groups is not None and count != n_groups:
        raise ValueError(f"{what}: {count} groups for {n_groups} matrices")
    return count


def _struct(groups: RowGroups, x, y, w, device) -> _lib.GroupedStruct:
    a = _lib.GroupedStruct()
    a.type = TYPES[x.dtype]
    a.groups, a.rows, a.k, a.n = groups.offsets.shape[0] - 1, x.shape[0], x.shape[1], y.shape[1]
    a.order, a.offsets = groups.rows.data_ptr(), groups.offsets.data_ptr()
    a.x, a.y, a.w = x.data_ptr(), y.data_ptr(), w.data_ptr()
    a.x_stride, a.y_stride = max(x.stride(0), x.shape[1]), max(y.stride(0), y.shape[1])
    a.w_group_stride, a.w_row_stride = w.stride(0), w.stride(1)
    a.status = _status_of(device).data_ptr()
    return a


def _rows_product(what: str, entry: str, source, weight, groups, out, transposed: bool):
    _matrix(what, "the input", source)
    _weights(what, "weight", weight)
    if source.dtype not in TYPES or weight.dtype != source.dtype:
        raise ValueError(f"{what}: input and weight must have the same type, float32, bfloat16 or float16")
    wide_in, wide_out = (weight.shape[2], weight.shape[1]) if transposed else (weight.shape[1], weight.shape[2])
    if source.shape[1] != wide_in:
        raise ValueError(f"{what}: rows of {source.shape[1]} values for matrices that take {wide_in}")
    if wide_in < 1 or wide_out < 1:
        raise ValueError(f"{what}: empty matrices")
    rows = source.shape[0]
    _groups(what, groups, rows, weight.shape[0])
    given = out is not None
    device = _on_device(what, source, weight, *groups, *((out,) if given else ()))
    if given:
        _matrix(what, "out", out, (rows, wide_out))
        if out.dtype != source.dtype:
            raise ValueError(f"{what}: out must have the input's type")
    with torch.cuda.device(device):
        if not given:
            out = torch.empty(rows, wide_out, dtype=source.dtype, device=device)
        if rows:
            x, y = (out, source) if transposed else (source, out)
            a = _struct(groups, x, y, weight, device)
            a.zero_rest = int(not given)
            _lib.check(getattr(_lib.load(), entry)(ctypes.byref(a), _lib.current_stream()), entry)
    return out


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, groups: RowGroups, out: torch.Tensor | None = None) -> torch.Tensor:
    """``y[r] = x[r] W[g(r)]``: x ``[rows, k]``, weight ``[groups, k, n]``, y ``[rows, n]`` of the same type."""
    return _rows_product("grouped_linear", "fmb_grouped_linear", x, weight, groups, out, False)


def grouped_linear_input_gradient(dy: torch.Tensor, weight: torch.Tensor, groups: RowGroups,
                                  out: torch.Tensor | None = None) -> torch.Tensor:
    """``dx[r] = dy[r] W[g(r)]^T``: the adjoint of ``grouped_linear`` in its input."""
    return _rows_product("grouped_linear_input_gradient", "fmb_grouped_input_gradient", dy, weight, groups, out, True)


def grouped_linear_weight_gradient(x: torch.Tensor, dy: torch.Tensor, groups: RowGroups, out: torch.Tensor | None = None,
                                   accumulate: bool = False) -> torch.Tensor:
    """``dW[g] = sum of x[r]^T dy[r]`` over the rows of g, float32 ``[groups, k, n]``; zero for a group without rows.
    ``accumulate=True`` adds to ``out``. The sums run in an order that depends on the sizes alone."""
    what = "grouped_linear_weight_gradient"
    _matrix(what, "x", x)
    _matrix(what, "dy", dy)
    if x.dtype not in TYPES or dy.dtype != x.dtype:
        raise ValueError(f"{what}: x and dy must have the same type, float32, bfloat16 or float16")
    if x.shape[0] != dy.shape[0]:
        raise ValueError(f"{what}: {x.shape[0]} rows of x for {dy.shape[0]} of dy")
    if x.shape[1] < 1 or dy.shape[1] < 1:
        raise ValueError(f"{what}: empty rows")
    count = _groups(what, groups, x.shape[0], None)
    shape = (count, x.shape[1], dy.shape[1])
    given = out is not None
    if accumulate and not given:
        raise ValueError(f"{what}: accumulate needs out")
    device = _on_device(what, x, dy, *groups, *((out,) if given else ()))
    if given:
        _weights(what, "out", out)
        if tuple(out.shape) != shape or out.dtype != torch.float32:
            raise ValueError(f"{what}: out must be float32 {shape}")
    with torch.cuda.device(device):
        if not given:
            out = torch.empty(shape, dtype=torch.float32, device=device)
        lib = _lib.load()
        a = _struct(groups, x, dy, out, device)
        a.accumulate = int(bool(accumulate))
        need = lib.fmb_grouped_scratch(ctypes.byref(a))
        scratch = torch.empty(need, dtype=torch.float32, device=device) if need else None
        a.scratch = scratch.data_ptr() if need else None
        _lib.check(lib.fmb_grouped_weight_gradient(ctypes.byref(a), _lib.current_stream()), "fmb_grouped_weight_gradient")
    return out


__all__ = ["RowGroups", "group_rows", "grouped_linear", "grouped_linear_input_gradient", "grouped_linear_weight_gradient",
           "check_status", "prepare_device", "MAX_GROUPS"]
