"""Refusals of the calls on held rows that need no GPU: there is no CPU path, and the C entries check what they are given."""
import ctypes

import pytest
import torch


def _lib():
    from fastmace_b200 import _lib, build
    build.build()
    return _lib, _lib.load()


def test_host_tensors_are_refused():
    from fastmace_b200 import checkpoints, grouped
    x = torch.zeros(4, 64)
    codes = torch.zeros(4, 64, dtype=torch.float8_e4m3fn)
    held = checkpoints.HeldRows(codes, torch.zeros(4, 2, dtype=torch.uint8), torch.float32)
    plan = grouped.RowGroups(torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    for call in (lambda: checkpoints.hold_rows(x), lambda: checkpoints.release_rows(held), lambda: checkpoints.gated_rows(x),
                 lambda: checkpoints.gated_rows_gradient(x, x[:, :32]), lambda: checkpoints.gated_rows_gradient(held._replace(parts=2), x[:, :32]),
                 lambda: checkpoints.held_weight_gradient(held, x, plan)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def _held(_lib, **changes):
    """A call whose every check passes; the pointers are never followed, each test breaks one field."""
    a = _lib.HeldStruct()
    a.type, a.rows, a.columns, a.parts = 1, 8, 64, 2
    a.x = a.codes = a.exponents = a.h = a.dh = a.du = 4096
    a.x_stride, a.h_stride, a.dh_stride, a.du_stride = 64, 64, 32, 64
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change", [dict(type=3), dict(rows=-1), dict(rows=(1 << 30) + 1), dict(columns=0), dict(columns=(1 << 20) + 2),
                                    dict(parts=0), dict(parts=3), dict(columns=63), dict(codes=None), dict(exponents=None)])
@pytest.mark.parametrize("entry", ["fmb_hold_rows", "fmb_release_rows", "fmb_gated_rows", "fmb_gated_rows_gradient"])
def test_held_entries_refuse(entry, change):
    mod, lib = _lib()
    assert getattr(lib, entry)(ctypes.byref(_held(mod, **change)), None) == 1          # FMB_ERR_ARG
    assert lib.fmb_last_error() and getattr(lib, entry)(None, None) == 1


@pytest.mark.parametrize("entry,change", [("fmb_hold_rows", dict(x=None)), ("fmb_hold_rows", dict(x_stride=63)),
                                          ("fmb_hold_rows", dict(codes=None, exponents=None)), ("fmb_release_rows", dict(h=None)),
                                          ("fmb_release_rows", dict(h_stride=63)), ("fmb_release_rows", dict(codes=None, exponents=None)),
                                          ("fmb_gated_rows", dict(x=None)), ("fmb_gated_rows", dict(h=None)), ("fmb_gated_rows", dict(parts=1)),
                                          ("fmb_gated_rows", dict(x_stride=63)), ("fmb_gated_rows", dict(h_stride=31)),
                                          ("fmb_gated_rows_gradient", dict()), ("fmb_gated_rows_gradient", dict(x=None, dh=None)),
                                          ("fmb_gated_rows_gradient", dict(x=None, du=None)), ("fmb_gated_rows_gradient", dict(x=None, parts=1)),
                                          ("fmb_gated_rows_gradient", dict(x=None, codes=None, exponents=None)),
                                          ("fmb_gated_rows_gradient", dict(x=None, dh_stride=31)), ("fmb_gated_rows_gradient", dict(x=None, du_stride=63)),
                                          ("fmb_gated_rows_gradient", dict(x=None, h_stride=31))])
def test_held_entries_refuse_what_they_need(entry, change):
    mod, lib = _lib()
    assert getattr(lib, entry)(ctypes.byref(_held(mod, **change)), None) == 1


@pytest.mark.parametrize("kind", [0, 1, 2])
def test_held_weight_gradient_entry_refuses(kind):
    mod, lib = _lib()

    def call(exponents=4096, **changes):
        a = mod.GroupedStruct()
        a.type, a.groups, a.rows, a.k, a.n = kind, 2, 8, 16, 24
        a.order = a.offsets = a.x = a.y = a.w = a.scratch = 4096
        a.x_stride, a.y_stride, a.w_row_stride, a.w_group_stride = 16, 24, 24, 24 * 16
        for name, value in changes.items():
            setattr(a, name, value)
        return lib.fmb_held_weight_gradient(ctypes.byref(a), exponents, None)

    for change in (dict(type=3), dict(groups=0), dict(k=0), dict(x=None), dict(w=None), dict(x_stride=24), dict(exponents=None), dict(scratch=None),
                   dict(scratch=4100)):
        assert call(**change) == 1, change
    assert lib.fmb_held_weight_gradient(None, 4096, None) == 1 and lib.fmb_held_weight_gradient_scratch(None) == 0
