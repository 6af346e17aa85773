"""Rows of a table by token -- the element embedding of an atom, or the vocabulary of a model of text -- and the table's gradient
(``csrc/embedding.cu``, ``csrc/grouping.cu``).

    y  = embedding(tokens, table, scale)                           # y[r]  = scale E[t(r)]
    order = sort_tokens(tokens, vocabulary)                        # once per batch of tokens
    dE = embedding_gradient(dy, order, vocabulary, scale)          # dE[v] = scale * sum of dy[r] over the rows of token v, fp32

``tokens``: int32 or int64, one per row. A token that is no row of the table (negative, as padding has it, or >= the vocabulary) gives
a row of zeros in an output the call allocates, leaves the row as it was in one that is given, and takes no part in a gradient. Table,
rows and ``dy``: float32, bfloat16 or float16, up to 2^30 rows and 2^20 columns, rows possibly further apart than they are long. The
product with ``scale`` is made in float32 and rounded once. The gradient is float32 whatever the rows' type, summed in float32 without atomics: the same call gives the
same bits. It is the whole table's, with zeros where a token has no rows, as ``optimiser.AdamW`` takes it; with ``accumulate`` the rows
of such tokens are not touched.

Calls run on the current stream of the operands' device and allocate their outputs and scratch from torch's allocator, so
they can be captured; a captured call may be replayed on other tokens. Nothing synchronises. There is no autograd and no CPU path.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .grouped import TYPES, _launch, _matrix, _on_device, _shares_memory, _written

MAX_VOCABULARY = _lib.MAX_VOCABULARY
MAX_ROWS, MAX_COLUMNS = 1 << 30, 1 << 20


def _empty(rows: int, columns: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """``torch.empty``, in two thirds of its time on the host."""
    return torch.empty_strided((rows, columns), (columns, 1), dtype=dtype, device=device)


def _scratch(size: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    return torch.empty_strided((size,), (1,), dtype=dtype, device=device)


def _limits(what: str, rows: int, columns: int, most: int = MAX_ROWS) -> None:
    if rows > most or columns > MAX_COLUMNS:
        raise ValueError(f"{what}: {rows} x {columns}, of {most} rows and {MAX_COLUMNS} columns at most")


class TokenOrder(NamedTuple):
    """``rows``: int32, the row numbers by token, in ascending order within a token, then the rows without one; ``keys``: int32, their
    tokens, the vocabulary's size for none."""
    rows: torch.Tensor
    keys: torch.Tensor


def _tokens(what: str, tokens: torch.Tensor) -> torch.Tensor:
    if tokens.dim() != 1 or tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: tokens must be one int32 or int64 per row")
    return tokens if tokens.shape[0] < 2 or tokens.stride(0) == 1 else tokens.contiguous()


def _vocabulary(what: str, size: int) -> int:
    if not 1 <= int(size) <= MAX_VOCABULARY:
        raise ValueError(f"{what}: a vocabulary of 1 to {MAX_VOCABULARY}")
    return int(size)


def sort_tokens(tokens: torch.Tensor, vocabulary: int) -> TokenOrder:
    """The rows by token, a stable order. Does not synchronise."""
    vocabulary = _vocabulary("sort_tokens", vocabulary)
    index = _on_device("sort_tokens", tokens)
    tokens = _tokens("sort_tokens", tokens)
    rows, lib, device = tokens.shape[0], _lib.load(), tokens.device
    out = TokenOrder(_scratch(rows, torch.int32, device), _scratch(rows, torch.int32, device))
    need = lib.fmb_sort_tokens_scratch(rows, vocabulary)
    scratch = _scratch(need, torch.int32, device) if need else None
    _lib.check(_launch(index, lib.fmb_sort_tokens, tokens.data_ptr(), tokens.element_size(), rows, vocabulary, out.rows.data_ptr(),
                       out.keys.data_ptr(), scratch.data_ptr() if need else None), "fmb_sort_tokens")
    return out


def embedding(tokens: torch.Tensor, table: torch.Tensor, scale: float = 1.0, out: torch.Tensor | None = None,
              dtype: torch.dtype | None = None) -> torch.Tensor:
    """``y[r] = scale E[t(r)]``: tokens ``[rows]``, table ``[vocabulary, width]``, y ``[rows, width]`` of the table's type, or of
    ``dtype`` (float32, bfloat16 or float16)."""
    what = "embedding"
    size, width, stride = _matrix(what, "table", table)
    vocabulary = _vocabulary(what, size)
    kind = TYPES.get(table.dtype)
    dtype = dtype if dtype is not None else out.dtype if out is not None else table.dtype
    if kind is None or dtype not in TYPES:
        raise ValueError(f"{what}: table and rows must be float32, bfloat16 or float16")
    _limits(what, tokens.shape[0] if tokens.dim() else 0, width)
    index = _on_device(what, tokens, table)
    tokens = _tokens(what, tokens)
    rows, given = tokens.shape[0], out is not None
    if given:
        out_stride = _matrix(what, "out", out, width, rows)[2]
        if out.dtype != dtype:
            raise ValueError(f"{what}: out must have the type asked for")
        _on_device(what, table, out)
        if _shares_memory(out, table) or _shares_memory(out, tokens):
            raise ValueError(f"{what}: out shares memory with an operand")
    else:
        out, out_stride = _empty(rows, width, dtype, table.device), width
    if rows:
        lib = _lib.load()
        a = _lib.EmbeddingStruct(kind, TYPES[dtype], rows, vocabulary, width, tokens.element_size(), not given, 0, float(scale),
                                 tokens.data_ptr(), None, table.data_ptr(), out.data_ptr(), stride, out_stride, None)
        _lib.check(_launch(index, lib.fmb_embedding, ctypes.byref(a)), "fmb_embedding")
        if given:
            _written(out)
    return out


def embedding_gradient(dy: torch.Tensor, order: TokenOrder, vocabulary: int, scale: float = 1.0, out: torch.Tensor | None = None,
                       accumulate: bool = False) -> torch.Tensor:
    """``dE[v] = scale * sum of dy[r]`` over the rows of token v: dy ``[rows, width]``, float32 ``[vocabulary, width]``.
    ``order``: as ``sort_tokens`` gives it for the same vocabulary. ``accumulate=True`` adds to ``out``."""
    what = "embedding_gradient"
    rows, width, stride = _matrix(what, "dy", dy)
    _limits(what, rows, width)
    vocabulary = _vocabulary(what, vocabulary)
    kind = TYPES.get(dy.dtype)
    if kind is None:
        raise ValueError(f"{what}: dy must be float32, bfloat16 or float16")
    for t in order:
        if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() or t.shape[0] != rows:
            raise ValueError(f"{what}: order must be as sort_tokens returns it, for {rows} rows")
    index = _on_device(what, dy, *order)
    given = out is not None
    if given:
        out_stride = _matrix(what, "out", out, width, vocabulary)[2]
        if out.dtype != torch.float32:
            raise ValueError(f"{what}: out must be float32")
        _on_device(what, dy, out)
        if any(_shares_memory(out, t) for t in (dy, *order)):
            raise ValueError(f"{what}: out shares memory with an operand")
    else:
        if accumulate:
            raise ValueError(f"{what}: accumulate needs out")
        out, out_stride = _empty(vocabulary, width, torch.float32, dy.device), width
    lib = _lib.load()
    a = _lib.EmbeddingStruct(kind, 0, rows, vocabulary, width, 4, 0, bool(accumulate), float(scale), order.keys.data_ptr(),
                             order.rows.data_ptr(), dy.data_ptr(), out.data_ptr(), stride, out_stride, None)
    need = lib.fmb_embedding_gradient_scratch(ctypes.byref(a))
    if need:
        scratch = _scratch(need, torch.float32, dy.device)
        a.scratch = scratch.data_ptr()
    _lib.check(_launch(index, lib.fmb_embedding_gradient, ctypes.byref(a)), "fmb_embedding_gradient")
    if given:
        _written(out)
    return out


__all__ = ["TokenOrder", "sort_tokens", "embedding", "embedding_gradient", "MAX_VOCABULARY"]
