"""Products with one matrix per group of rows -- the species-dependent linear of an interaction (``l{t}.skip.{l}``), or the
experts of a layer -- with any number of rows per group, and their gradients (``csrc/grouping.cu``, ``csrc/grouped.cu``).

    groups = group_rows(species, n_species)                         # rows by group, once per set of atoms
    y  = grouped_linear(x, weight, groups)                          # y[r]  = x[r] W[g(r)]
    dx = grouped_linear_input_gradient(dy, weight, groups)          # dx[r] = dy[r] W[g(r)]^T
    dw = grouped_linear_weight_gradient(x, dy, groups)              # dW[g] = sum over its rows of x[r]^T dy[r], fp32

Rows keep their places: row r of ``y`` belongs to row r of ``x`` whatever the order of the groups. ``x`` and ``dy`` may be
views whose rows are further apart than they are long (a component of ``[atom][component][channel]`` features), ``weight``
any ``[groups, k, n]`` view with contiguous columns (``w["l1.skip.0"].permute(1, 0, 2)``). Types: float32, bfloat16, float16,
the same for all operands of a call; sums are in float32 at least, the weight gradient is float32 whatever the operands'. float32
operands keep their 24 bits from 2^-110 on, and less of smaller ones: what lies below 2^-133 is lost. A row of no group (key negative or >= the number of groups) is zero in an output the call
allocates, left as it was in one that is given, and takes no part in a weight gradient.

Calls run on the current stream of the operands' device and allocate their outputs and scratch from torch's allocator, so
they can be captured, after one call of the same kind outside a capture. The groups are read on the device: nothing synchronises,
and a captured call may be replayed on other groups. A kernel that gives up waiting raises nothing by itself: ``check_status``.
There is no autograd and no CPU path.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib

MAX_GROUPS = _lib.MAX_GROUPS
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MOST = 2 ** 31 - 1                            # what an entry's 32 bits hold; a larger number would lose its upper ones on the way


class RowGroups(NamedTuple):
    """``rows``: int32, the row numbers of group 0, then of group 1, ..., then of the rows without a group; ``offsets``:
    int32 ``[groups + 1]``, where each group starts."""
    rows: torch.Tensor
    offsets: torch.Tensor


_status: dict[int, torch.Tensor] = {}         # a status word per device, read by check_status


def _status_pointer(index: int) -> int:
    word = _status.get(index)
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            raise _lib.Fmb200Error("call grouped.prepare_device() before capturing the first grouped product of a device")
        word = torch.zeros((), dtype=torch.int32, device=torch.device("cuda", index))
        torch.cuda.current_stream(word.device).synchronize()       # other streams may use it from here on
        _status[index] = word
    return word.data_ptr()


def _index(device) -> int:
    device = torch.device(device)
    return device.index if device.index is not None else torch.cuda.current_device()


def prepare_device(device="cuda") -> None:
    """Makes the device's status word; needed only where the first product on a device would be a captured one."""
    _status_pointer(_index(device))


def check_status(device="cuda") -> None:
    """Raises if a grouped product on ``device`` gave up waiting since the last check (synchronises)."""
    word = _status.get(_index(device))
    if word is not None and int(word.item()) & _lib.STATUS_TENSOR_TIMEOUT:
        word.zero_()
        raise _lib.Fmb200Error("a tensor-core kernel gave up waiting (FMB_STATUS_TENSOR_TIMEOUT)")


def _on_device(what: str, *tensors: torch.Tensor) -> int:
    index = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != index or index < 0:
            raise ValueError(f"{what}: the operands must be CUDA tensors on one device, there is no CPU path")
    return index


def _launch(index: int, call, *arguments):
    """``call(*arguments, stream)`` with the device current and its current stream."""
    stream = torch._C._cuda_getCurrentRawStream(index)       # what torch.cuda.current_stream holds, a twentieth of its time
    if torch.cuda.current_device() == index:
        return call(*arguments, stream)
    with torch.cuda.device(index):
        return call(*arguments, stream)


def _written(out: torch.Tensor) -> None:
    """Tells autograd that a given output has changed in place (inference tensors have no version to count)."""
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)


def group_rows(keys: torch.Tensor, n_groups: int) -> RowGroups:
    """Rows by group for ``keys`` (int32 or int64, one per row): a stable order, so equal keys keep the order of their rows.
    1 to 1,024 groups. Does not synchronise."""
    if keys.dim() != 1 or keys.dtype not in (torch.int32, torch.int64):
        raise ValueError("group_rows: keys must be one int32 or int64 per row")
    if not 1 <= int(n_groups) <= MAX_GROUPS:
        raise ValueError(f"group_rows: 1 to {MAX_GROUPS} groups")
    index = _on_device("group_rows", keys)
    if keys.shape[0] > 1 and keys.stride(0) != 1:
        keys = keys.contiguous()
    rows, lib, device = keys.shape[0], _lib.load(), keys.device
    out = RowGroups(torch.empty(rows, dtype=torch.int32, device=device),
                    torch.empty(int(n_groups) + 1, dtype=torch.int32, device=device))
    need = lib.fmb_group_rows_scratch(rows, int(n_groups))
    scratch = torch.empty(need, dtype=torch.int32, device=device) if need else None
    _lib.check(_launch(index, lib.fmb_group_rows, keys.data_ptr(), keys.element_size(), rows, int(n_groups), out.rows.data_ptr(),
                       out.offsets.data_ptr(), scratch.data_ptr() if need else None), "fmb_group_rows")
    return out


def _matrix(what: str, name: str, t: torch.Tensor, columns: int | None = None, rows: int | None = None):
    """(rows, columns, row stride) of a matrix with contiguous rows."""
    if t.dim() != 2:
        raise ValueError(f"{what}: {name} must be a matrix, got {tuple(t.shape)}")
    (m, n), (far, near) = t.shape, t.stride()
    if (columns is not None and n != columns) or (rows is not None and m != rows):
        raise ValueError(f"{what}: {name} is {m} x {n}, expected {m if rows is None else rows} x {n if columns is None else columns}")
    if n < 1:
        raise ValueError(f"{what}: {name} has empty rows")
    if m > MOST or n > MOST:
        raise ValueError(f"{what}: {name} is {m} x {n}, of {MOST} rows and columns at most")
    if (n > 1 and near != 1) or (m > 1 and far < n):
        raise ValueError(f"{what}: {name} must have contiguous rows that do not overlap")
    return m, n, far if m > 1 else n


def _shares_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors may have elements in common: false for ones that lie apart, and for rows of the same distance that lie
    side by side (two components of one array of features)."""
    size_a, size_b = a.element_size(), b.element_size()
    reach = lambda t: sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1  # noqa: E731
    if not a.numel() or not b.numel():
        return False
    at_a, at_b = a.data_ptr(), b.data_ptr()
    if at_a + size_a * reach(a) <= at_b or at_b + size_b * reach(b) <= at_a:
        return False
    if a.dim() == b.dim() == 2 and size_a == size_b and a.stride(0) == b.stride(0) and (at_b - at_a) % size_a == 0:
        stride = a.stride(0)
        apart = (at_b - at_a) // size_a % stride if stride else 0
        return not (a.shape[1] <= apart and apart + b.shape[1] <= stride)
    return True


def _weights(what: str, name: str, t: torch.Tensor):
    """(groups, k, n, group stride, row stride) of the matrices of all groups."""
    if t.dim() != 3:
        raise ValueError(f"{what}: {name} must be [groups, k, n], got {tuple(t.shape)}")
    (g, k, n), (between, far, near) = t.shape, t.stride()
    if n > 1 and near != 1:
        raise ValueError(f"{what}: the columns of {name} must be contiguous")
    if k > MOST or n > MOST:
        raise ValueError(f"{what}: {name} is {k} x {n}, of {MOST} rows and columns at most")
    return g, k, n, between, far


def _groups(what: str, groups: RowGroups, rows: int, n_groups: int | None = None) -> int:
    order, offsets = groups
    if order.dtype != torch.int32 or offsets.dtype != torch.int32 or order.dim() != 1 or offsets.dim() != 1 or \
            not order.is_contiguous() or not offsets.is_contiguous():
        raise ValueError(f"{what}: groups must be as group_rows returns them")
    count = offsets.shape[0] - 1
    if order.shape[0] != rows or not 1 <= count <= MAX_GROUPS or (n_groups is not None and count != n_groups):
        raise ValueError(f"{what}: {count} groups of {order.shape[0]} rows, expected {n_groups or f'1 to {MAX_GROUPS}'} of {rows}")
    return count


def _rows_product(what: str, entry: str, source, weight, groups, out, transposed: bool):
    count, k, n, w_group, w_row = _weights(what, "weight", weight)
    rows, width, stride = _matrix(what, "the input", source, n if transposed else k)
    dtype = source.dtype
    kind = TYPES.get(dtype)
    if kind is None or weight.dtype != dtype:
        raise ValueError(f"{what}: input and weight must have the same type, float32, bfloat16 or float16")
    if k < 1 or n < 1:
        raise ValueError(f"{what}: empty matrices")
    _groups(what, groups, rows, count)
    index = _on_device(what, source, weight, *groups)
    wide_out = k if transposed else n
    given = out is not None
    if given:
        out_stride = _matrix(what, "out", out, wide_out, rows)[2]
        if out.dtype != dtype:
            raise ValueError(f"{what}: out must have the input's type")
        _on_device(what, source, out)
        if _shares_memory(out, source) or _shares_memory(out, weight):
            raise ValueError(f"{what}: out shares memory with an operand")
    else:
        out, out_stride = source.new_empty((rows, wide_out)), wide_out
    if rows:
        lib, here, there = _lib.load(), source.data_ptr(), out.data_ptr()
        x, y, x_stride, y_stride = (there, here, out_stride, stride) if transposed else (here, there, stride, out_stride)
        a = _lib.GroupedStruct(kind, count, rows, k, n, not given, 0, 0, groups[0].data_ptr(), groups[1].data_ptr(), x, y,
                               weight.data_ptr(), x_stride, y_stride, w_row, w_group, None, _status_pointer(index))
        call = ctypes.byref(a)
        need = lib.fmb_grouped_scratch(call, int(transposed))
        if need:
            scratch = torch.empty(need, dtype=torch.float32, device=source.device)
            a.scratch = scratch.data_ptr()
        _lib.check(_launch(index, getattr(lib, entry), call), entry)
        if given:
            _written(out)
    return out


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, groups: RowGroups, out: torch.Tensor | None = None) -> torch.Tensor:
    """``y[r] = x[r] W[g(r)]``: x ``[rows, k]``, weight ``[groups, k, n]``, y ``[rows, n]`` of the same type."""
    return _rows_product("grouped_linear", "fmb_grouped_linear", x, weight, groups, out, False)


def grouped_linear_input_gradient(dy: torch.Tensor, weight: torch.Tensor, groups: RowGroups,
                                  out: torch.Tensor | None = None) -> torch.Tensor:
    """``dx[r] = dy[r] W[g(r)]^T``: the adjoint of ``grouped_linear`` in its input."""
    return _rows_product("grouped_linear_input_gradient", "fmb_grouped_input_gradient", dy, weight, groups, out, True)


def _weight_gradient(what: str, x: torch.Tensor, x_stride: int, dtype: torch.dtype, dy: torch.Tensor, groups: RowGroups,
                     out: torch.Tensor | None, accumulate: bool, exponents: torch.Tensor | None = None) -> torch.Tensor:
    """The weight gradient of rows x, or of the codes x and exponents of rows of type ``dtype`` that are held in 8 bits."""
    rows, k = x.shape
    _, n, y_stride = _matrix(what, "dy", dy, rows=rows)
    kind = TYPES.get(dtype)
    if kind is None or dy.dtype != dtype:
        raise ValueError(f"{what}: x and dy must have the same type, float32, bfloat16 or float16")
    count = _groups(what, groups, rows)
    index = _on_device(what, x, dy, *groups)
    given = out is not None
    if not given:
        if accumulate:
            raise ValueError(f"{what}: accumulate needs out")
        out = torch.empty((count, k, n), dtype=torch.float32, device=x.device)
    elif out.dtype != torch.float32 or tuple(out.shape) != (count, k, n):
        raise ValueError(f"{what}: out must be float32 {(count, k, n)}")
    else:
        _on_device(what, x, out)
        if _shares_memory(out, x) or _shares_memory(out, dy) or (exponents is not None and _shares_memory(out, exponents)):
            raise ValueError(f"{what}: out shares memory with an operand")
    _, _, _, w_group, w_row = _weights(what, "out", out)
    far, near, inner = (max(w_row, w_group), min(w_row, w_group), k if w_group >= w_row else count)
    if k > 1 and count > 1 and (near < n or far < (inner - 1) * near + n) or k > 1 and count == 1 and w_row < n or \
            k == 1 and count > 1 and w_group < n:
        raise ValueError(f"{what}: the matrices of out overlap")
    lib = _lib.load()
    a = _lib.GroupedStruct(kind, count, rows, k, n, 0, bool(accumulate), 0, groups[0].data_ptr(), groups[1].data_ptr(), x.data_ptr(),
                           dy.data_ptr(), out.data_ptr(), x_stride, y_stride, w_row, w_group, None, _status_pointer(index))
    call = ctypes.byref(a)
    need = lib.fmb_grouped_scratch(call, 2) if exponents is None else lib.fmb_held_weight_gradient_scratch(call)
    if need:
        scratch = torch.empty(need, dtype=torch.float32, device=x.device)
        a.scratch = scratch.data_ptr()
    if exponents is None:
        _lib.check(_launch(index, lib.fmb_grouped_weight_gradient, call), "fmb_grouped_weight_gradient")
    else:
        _lib.check(_launch(index, lib.fmb_held_weight_gradient, call, exponents.data_ptr()), "fmb_held_weight_gradient")
    if given:
        _written(out)
    return out


def grouped_linear_weight_gradient(x: torch.Tensor, dy: torch.Tensor, groups: RowGroups, out: torch.Tensor | None = None,
                                   accumulate: bool = False) -> torch.Tensor:
    """``dW[g] = sum of x[r]^T dy[r]`` over the rows of g, float32 ``[groups, k, n]``; zero for a group without rows.
    ``accumulate=True`` adds to ``out``. The sums run in an order that depends on the sizes alone. Rows x that are held in 8 bits:
    ``checkpoints.held_weight_gradient``."""
    what = "grouped_linear_weight_gradient"
    stride = _matrix(what, "x", x)[2]
    return _weight_gradient(what, x, stride, x.dtype, dy, groups, out, accumulate)


__all__ = ["RowGroups", "group_rows", "grouped_linear", "grouped_linear_input_gradient", "grouped_linear_weight_gradient",
           "check_status", "prepare_device", "MAX_GROUPS"]
