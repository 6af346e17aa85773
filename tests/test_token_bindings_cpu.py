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
