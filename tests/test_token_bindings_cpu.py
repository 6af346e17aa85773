"""What the entries of embedding rows, held rows and experts are told and say, as far as that needs no GPU."""
import ctypes
import os
import re

import pytest
import torch
from conftest import ROOT


def _lib():
    from fastmace_b200 import _lib, build
    build.build()
    return _lib, _lib.load()


def test_results_of_entries_have_the_type_that_the_header_declares():
    mod, lib = _lib()
    header = open(os.path.join(ROOT, "include", "fmb200.h")).read()
    declared = dict((name, kind.strip()) for kind, name in re.findall(r"FMB_API\s+([\w\s]+?[\s\*]+)(fmb_\w+)\s*\(", header))
    assert set(declared) == set(mod.EXPORTS)
    kinds = {"int": ctypes.c_int, "long long": ctypes.c_longlong, "const char*": ctypes.c_char_p}
    for name, kind in declared.items():
        assert getattr(lib, name).restype is kinds[kind], name


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("rows,width", [(1, 1), (300, 515), (9000, 129), (65_536, 1024), (884_736, 128), (3_000_000, 8), (100_000, 4097)])
def test_scratch_of_the_embedding_gradient_goes_by_sizes_and_type(kind, rows, width):
    """A host may ask for it with rows in one place and call with rows in another."""
    mod, lib = _lib()

    def need(source, stride):
        a = mod.EmbeddingStruct()
        a.type, a.rows, a.vocabulary, a.width, a.token_bytes, a.scale = kind, rows, 7, width, 4, 1.0
        a.tokens = a.order = a.out = 4096
        a.source, a.source_stride, a.out_stride = source, stride, width
        return lib.fmb_embedding_gradient_scratch(ctypes.byref(a))

    wide = (width + 7) // 8 * 8
    assert len({need(source, stride) for source in (None, 4096, 4098, 4104) for stride in (width, wide, wide + 1)}) == 1


@pytest.mark.parametrize("rows", [2 ** 32 + 5, 2 ** 31, 2 ** 30 + 1])
def test_counts_past_what_an_entry_takes_are_refused(rows):
    """A count goes to an entry in 32 bits: 2^32 + 5 rows would be 5 there, and the others left as they are."""
    from fastmace_b200 import checkpoints, embedding, experts, grouped
    bf16 = torch.bfloat16

    def of(*shape, dtype=bf16):
        return torch.empty(shape, dtype=dtype, device="meta")            # (sizes without memory; refused before a device is asked for)

    held = [checkpoints.HeldRows(of(rows, 8, dtype=torch.float8_e4m3fn), of(rows, parts, dtype=torch.uint8), bf16, parts) for parts in (1, 2)]
    tokens, order = of(rows, dtype=torch.int32), embedding.TokenOrder(of(rows, dtype=torch.int32), of(rows, dtype=torch.int32))
    plan = grouped.RowGroups(of(rows, dtype=torch.int32), of(3, dtype=torch.int32))
    calls = [lambda: embedding.embedding(tokens, of(3, 8)), lambda: embedding.embedding_gradient(of(rows, 8), order, 3),
             lambda: checkpoints.hold_rows(of(rows, 8)), lambda: checkpoints.release_rows(held[0]), lambda: checkpoints.gated_rows(of(rows, 8)),
             lambda: checkpoints.gated_rows_gradient(held[1], of(rows, 4)), lambda: checkpoints.gated_rows_gradient(of(rows, 8), of(rows, 4)),
             lambda: checkpoints.held_weight_gradient(held[0], of(rows, 4), plan), lambda: experts.route_rows(of(rows, 8), of(8, 4), 2)]
    if rows > 2 ** 31 - 1:
        calls += [lambda: grouped.grouped_linear(of(rows, 8), of(2, 8, 4), plan), lambda: grouped.grouped_linear_input_gradient(of(rows, 4), of(2, 8, 4), plan),
                  lambda: grouped.grouped_linear_weight_gradient(of(rows, 8), of(rows, 4), plan), lambda: grouped.grouped_linear(of(2, rows), of(2, rows, 4), plan)]
    for call in calls:
        with pytest.raises(ValueError, match="at most"):
            call()
    with pytest.raises(ValueError, match="at most"):
        experts.route_rows(of((1 << 24) + 1, 8), of(8, 4), 2)
    for call in (lambda: embedding.embedding(of(4, dtype=torch.int32), of(3, (1 << 20) + 1)), lambda: checkpoints.hold_rows(of(4, (1 << 20) + 1)),
                 lambda: checkpoints.gated_rows(of(4, (1 << 20) + 2)), lambda: experts.route_rows(of(4, (1 << 20) + 1), of((1 << 20) + 1, 4), 2)):
        with pytest.raises(ValueError, match="at most"):
            call()
