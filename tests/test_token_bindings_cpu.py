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
