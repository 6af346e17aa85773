"""Refusals of the training operators that need no GPU: there is no CPU path, and the C entries check what they are given."""
import ctypes

import pytest
import torch


def _lib():
    from fastmace_b200 import _lib, build
    build.build()
    return _lib, _lib.load()


def test_host_tensors_are_refused():
    from fastmace_b200 import grouped
    from fastmace_b200.optimiser import AdamW
    x, w = torch.zeros(4, 8), torch.zeros(2, 8, 8)
    plan = grouped.RowGroups(torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    for call in (lambda: grouped.grouped_linear(x, w, plan), lambda: grouped.grouped_linear_input_gradient(x, w, plan),
                 lambda: grouped.grouped_linear_weight_gradient(x, x, plan),
                 lambda: grouped.group_rows(torch.zeros(4, dtype=torch.int32), 2), lambda: AdamW([x])):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def _grouped(_lib, **changes):
    """A call whose every check passes; the pointers are never followed, each test breaks one field."""
    a = _lib.GroupedStruct()
    a.type, a.groups, a.rows, a.k, a.n = 1, 2, 8, 16, 24
    a.order = a.offsets = a.x = a.y = a.w = a.scratch = 4096
    a.x_stride, a.y_stride, a.w_row_stride, a.w_group_stride = 16, 24, 24, 24 * 16
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change", [dict(type=3), dict(groups=0), dict(groups=1025), dict(rows=-1), dict(k=0), dict(n=0),
                                    dict(offsets=None), dict(order=None), dict(x=None), dict(y=None), dict(w=None),
                                    dict(x_stride=15), dict(y_stride=23)])
@pytest.mark.parametrize("entry", ["fmb_grouped_linear", "fmb_grouped_input_gradient", "fmb_grouped_weight_gradient"])
def test_grouped_entries_refuse(entry, change):
    mod, lib = _lib()
    assert getattr(lib, entry)(ctypes.byref(_grouped(mod, **change)), None) == 1          # FMB_ERR_ARG
    assert lib.fmb_last_error()
    assert getattr(lib, entry)(None, None) == 1


def test_group_rows_refuses():
    mod, lib = _lib()
    good = dict(keys=4096, key_bytes=4, rows=9000, groups=3, order=4096, offsets=4096, scratch=4096)
    for change in (dict(keys=None), dict(key_bytes=2), dict(rows=-1), dict(rows=1 << 31), dict(groups=0), dict(groups=1025),
                   dict(order=None), dict(offsets=None), dict(scratch=None)):
        assert lib.fmb_group_rows(*{**good, **change}.values(), None) == 1, change


def test_adamw_entry_refuses():
    mod, lib = _lib()

    def call(tensor=None, count=1, **changes):
        a = mod.AdamwStruct()
        a.moment_bits, a.grad_type, a.copy_type = 8, 0, 1
        a.lr, a.beta1, a.beta2, a.eps = 1e-3, 0.9, 0.999, 1e-8
        a.m = a.v = a.m_scale = a.v_scale = a.state = 4096
        for name, value in changes.items():
            setattr(a, name, value)
        t = (mod.AdamwTensorStruct * 1)()
        t[0].p, t[0].g, t[0].copy, t[0].values, t[0].block = 4096, 4096, 4096, 100, 0
        for name, value in (tensor or {}).items():
            setattr(t[0], name, value)
        return lib.fmb_adamw_step(ctypes.byref(a), t, count, None)

    for change in (dict(moment_bits=16), dict(grad_type=5), dict(m=None), dict(v=None), dict(state=None), dict(m_scale=None),
                   dict(m=4100), dict(beta1=1.0), dict(beta2=-0.1), dict(count=-1), dict(copy_type=0), dict(tensor=dict(p=None)),
                   dict(tensor=dict(p=4097)), dict(tensor=dict(values=-1)), dict(tensor=dict(block=-1)), dict(tensor=dict(copy=4097))):
        assert call(**change) == 1, change
    assert call(tensor=dict(g=None)) == 0 and call(count=0) == 0 and call(tensor=dict(values=0)) == 0


def test_what_shares_memory():
    from fastmace_b200.grouped import _shares_memory
    nodes = torch.zeros(10, 4, 16)
    assert _shares_memory(nodes[:, 1], nodes[:, 1]) and _shares_memory(nodes[:, 1], nodes[:, 1, 8:])
    assert not _shares_memory(nodes[:, 0], nodes[:, 1]) and not _shares_memory(nodes[:, 3], nodes[:, 0])
    assert not _shares_memory(nodes[:, 1, :8], nodes[:, 1, 8:]) and _shares_memory(nodes[:, 1, :9], nodes[:, 1, 8:])
    assert _shares_memory(nodes[:, 1], nodes.view(-1)[8:168].view(10, 16))
    assert not _shares_memory(nodes[:5, 1], nodes[5:, 1]) and not _shares_memory(nodes[:, 0], torch.zeros(10, 16))
    assert not _shares_memory(nodes[:0, 1], nodes[:, 1])
    # a row that goes round the end of the distance between rows
    wide = torch.zeros(200)
    assert _shares_memory(wide.as_strided((5, 10), (16, 1), 0), wide.as_strided((5, 10), (16, 1), 12))
    assert _shares_memory(wide[:64].view(8, 8), wide[8:72].view(2, 4, 8))
    assert _shares_memory(wide[:64].view(8, 8), wide[:64].view(torch.float16).view(8, 16))


@pytest.mark.parametrize("change", [dict(lr=float("nan")), dict(lr=float("inf")), dict(eps=float("nan")), dict(weight_decay=float("nan")),
                                    dict(betas=(float("nan"), 0.9)), dict(betas=(0.9, float("nan"))), dict(weight_decay=-1.0)])
def test_constants_that_are_no_numbers_are_refused(change):
    from fastmace_b200.optimiser import AdamW
    with pytest.raises(ValueError, match="finite|betas"):
        AdamW([torch.zeros(4)], **change)


def test_random_rounding_is_of_8_bit_moments():
    from fastmace_b200.optimiser import AdamW
    for change in (dict(rounding="random"), dict(rounding="down", state_bits=8), dict(rounding="random", state_bits=8, seed=-1),
                   dict(rounding="random", state_bits=8, seed=2 ** 31 - 1)):
        with pytest.raises(ValueError, match="rounding|seed"):
            AdamW([torch.zeros(4)], **change)
    mod, lib = _lib()
    a = mod.AdamwStruct()
    a.moment_bits, a.copy_type, a.beta1, a.beta2, a.random = 32, 1, 0.9, 0.999, 1
    a.m = a.v = a.state = 4096
    t = (mod.AdamwTensorStruct * 1)()
    assert lib.fmb_adamw_step(ctypes.byref(a), t, 1, None) == 1 and b"random" in lib.fmb_last_error()
    a.random = 0
    assert lib.fmb_adamw_step(ctypes.byref(a), t, 1, None) == 0
