"""Refusals of the embedding calls that need no GPU: there is no CPU path, and the C entries check what they are given."""
import ctypes

import pytest
import torch


def _lib():
    from fastmace_b200 import _lib, build
    build.build()
    return _lib, _lib.load()


def test_host_tensors_are_refused():
    from fastmace_b200 import embedding
    t, table = torch.zeros(4, dtype=torch.int32), torch.zeros(3, 8)
    order = embedding.TokenOrder(t, t)
    for call in (lambda: embedding.sort_tokens(t, 3), lambda: embedding.embedding(t, table),
                 lambda: embedding.embedding_gradient(torch.zeros(4, 8), order, 3)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def _embedding(_lib, **changes):
    """A call whose every check passes; the pointers are never followed, each test breaks one field."""
    a = _lib.EmbeddingStruct()
    a.type, a.out_type, a.rows, a.vocabulary, a.width, a.token_bytes, a.scale = 1, 0, 8000, 5, 16, 4, 1.0
    a.tokens = a.order = a.source = a.out = a.scratch = 4096
    a.source_stride, a.out_stride = 16, 16
    for name, value in changes.items():
        setattr(a, name, value)
    return a


SHARED = [dict(type=3), dict(type=-1), dict(rows=-1), dict(rows=(1 << 30) + 1), dict(vocabulary=0), dict(vocabulary=1 << 20), dict(width=0),
          dict(width=(1 << 20) + 1), dict(tokens=None), dict(source=None), dict(out=None), dict(source_stride=15), dict(out_stride=15)]


@pytest.mark.parametrize("change", SHARED + [dict(out_type=3), dict(token_bytes=2)])
def test_lookup_entry_refuses(change):
    mod, lib = _lib()
    assert lib.fmb_embedding(ctypes.byref(_embedding(mod, **change)), None) == 1          # FMB_ERR_ARG
    assert lib.fmb_last_error() and lib.fmb_embedding(None, None) == 1


@pytest.mark.parametrize("change", SHARED + [dict(order=None), dict(scratch=None), dict(scratch=4104)])
def test_gradient_entry_refuses(change):
    mod, lib = _lib()
    assert lib.fmb_embedding_gradient(ctypes.byref(_embedding(mod, **change)), None) == 1
    assert lib.fmb_last_error() and lib.fmb_embedding_gradient(None, None) == 1 and lib.fmb_embedding_gradient_scratch(None) == 0


def test_sort_tokens_refuses():
    mod, lib = _lib()
    good = dict(tokens=4096, token_bytes=4, rows=9000, vocabulary=3, order=4096, keys=4096, scratch=4096)
    for change in (dict(tokens=None), dict(token_bytes=2), dict(rows=-1), dict(rows=1 << 31), dict(vocabulary=0), dict(vocabulary=1 << 20),
                   dict(order=None), dict(keys=None), dict(scratch=None)):
        assert lib.fmb_sort_tokens(*{**good, **change}.values(), None) == 1, change
    assert lib.fmb_sort_tokens(*{**good, "rows": 0, "tokens": None}.values(), None) == 0


def test_scratch_covers_both_passes():
    mod, lib = _lib()
    for rows in (1, 8192, 8193, 100_000, 1 << 30):
        for vocabulary in (1, 1024, 1025, 4095, 4096, 100_003, (1 << 20) - 1):
            low = 0 if vocabulary <= 1024 else (vocabulary.bit_length() + 1) // 2
            widths = [vocabulary + 1] if not low else [1 << low, (vocabulary >> low) + 1]
            assert max(widths) <= 1025                     # what a table in shared memory holds
            per_cta = 2048 if rows <= 148 * 8 * 2048 else 8192
            tables = (-(-rows // per_cta) + 1) * max(widths)
            assert lib.fmb_sort_tokens_scratch(rows, vocabulary) == (0 if rows <= 8192 else tables + (rows if low else 0))
