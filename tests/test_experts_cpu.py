"""Refusals of the expert layer's calls that need no GPU: there is no CPU path, and the C entries check what they are given."""
import ctypes

import pytest
import torch


def _lib():
    from fastmace_b200 import _lib, build
    build.build()
    return _lib, _lib.load()


def test_host_tensors_are_refused():
    from fastmace_b200 import experts
    x = torch.zeros(4, 16)
    routes = experts.Routes(torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2))
    for call in (lambda: experts.route_rows(x, torch.zeros(16, 3), 2),
                 lambda: experts.expert_layer(x, torch.zeros(3, 16, 8), torch.zeros(3, 4, 16), routes)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def _filled(struct, values, changes):
    for name, kind in struct._fields_:
        if kind is ctypes.c_void_p:
            setattr(struct, name, 4096)
    for name, value in {**values, **changes}.items():
        setattr(struct, name, value)
    return struct


@pytest.mark.parametrize("change", [dict(type=3), dict(type=-1), dict(tokens=-1), dict(tokens=(1 << 24) + 1), dict(width=0), dict(experts=0),
                                    dict(experts=1025), dict(top=0), dict(top=17), dict(top=5), dict(x=None), dict(router=None), dict(chosen=None),
                                    dict(weights=None), dict(x_stride=15), dict(router_stride=3)])
def test_route_entry_refuses(change):
    mod, lib = _lib()
    a = _filled(mod.RouteStruct(), dict(type=1, tokens=8, width=16, experts=4, top=2, x_stride=16, router_stride=4), change)
    assert lib.fmb_route_rows(ctypes.byref(a), None) == 1 and lib.fmb_last_error() and lib.fmb_route_rows(None, None) == 1


@pytest.mark.parametrize("change", [dict(type=3), dict(type=-1), dict(tokens=-1), dict(tokens=129), dict(width=0), dict(width=(1 << 17) + 1),
                                    dict(inner=0), dict(inner=(1 << 17) + 1), dict(experts=0), dict(experts=1025), dict(top=0), dict(top=17), dict(x=None),
                                    dict(w_up=None), dict(w_down=None), dict(chosen=None), dict(weights=None), dict(y=None), dict(scratch=None),
                                    dict(scratch=4104), dict(x_stride=15), dict(y_stride=15)])
def test_layer_entry_refuses(change):
    mod, lib = _lib()
    a = _filled(mod.ExpertsStruct(), dict(type=1, tokens=8, experts=4, top=2, width=16, inner=24, x_stride=16, y_stride=16, up_group_stride=768,
                                          up_row_stride=48, down_group_stride=384, down_row_stride=16), change)
    assert lib.fmb_expert_layer(ctypes.byref(a), None) == 1 and lib.fmb_last_error()
    assert lib.fmb_expert_layer(None, None) == 1 and lib.fmb_expert_layer_scratch(None) == 0
