"""The C entries of attention, the bias of relative positions and dropout: every declared symbol is exported and bound, and what they
refuse before any launch."""
import ctypes
import os
import re

import pytest

from bit_reproducible_training_amd import _lib

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD = 1


def test_library_exports_every_declared_symbol():
    names = set()
    for header in ("repro_attention.h", "repro_dropout.h"):
        with open(os.path.join(REPO, "include", header)) as f:
            text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
        names |= set(re.findall(r"\b(rg_[a-z0-9_]+)\s*\(", text))
    assert names and names == set(_lib._SEQUENCE_SIGNATURES)
    for name in names:
        assert hasattr(_lib.lib, name), name


def config(**change):
    c = _lib.rg_attention_config()
    _lib.lib.rg_attention_config_init(ctypes.byref(c))
    c.B, c.Tq, c.Tk, c.H, c.KVH, c.D = 2, 3, 5, 4, 2, 8
    for n, v in change.items():
        setattr(c, n, v)
    return c


def test_defaults():
    c = _lib.rg_attention_config()
    _lib.lib.rg_attention_config_init(ctypes.byref(c))
    assert (c.B, c.Tq, c.Tk, c.H, c.KVH, c.D, c.causal, c.scale, c.dropout) == (1, 0, 0, 1, 1, 0, 0, 1.0, 0.0)


@pytest.mark.parametrize("change", [dict(B=-1), dict(Tq=-1), dict(Tk=2 ** 22 + 1), dict(H=0), dict(KVH=3), dict(D=0), dict(D=129),
                                    dict(scale=float("inf")), dict(dropout=1.0), dict(dropout=float("nan")), dict(B=2 ** 20),
                                    dict(q_stride=(ctypes.c_longlong * 3)(-1, 0, 0))])
def test_attention_refuses_bad_sizes(change):
    n, c = ctypes.c_size_t(), config(**change)
    assert _lib.lib.rg_attention_workspace(ctypes.byref(c), 0, ctypes.byref(n)) == BAD
    assert _lib.lib.rg_attention_grad_workspace(ctypes.byref(c), 0, ctypes.byref(n)) == BAD


def test_attention_refuses_bad_pointers():
    f, c = _lib.lib.rg_attention_fp32, config()
    good = [64, 64, 64, None, None, None, None, None, 64, None, None]  # addresses that are never read
    for at, bad in ((0, None), (1, None), (2, None), (8, None), (0, 66), (8, 66), (3, 68), (4, 68), (9, 68), (6, 68), (7, 68)):
        args = list(good)
        args[at] = bad
        assert f(ctypes.byref(c), *args, 0, None) == BAD, (at, bad)
    assert f(None, *good, 0, None) == BAD
    g = _lib.lib.rg_attention_grad_fp32
    good = [64, 64, 64, 64, None, None, None, None, 64, 64, 64, 64, 64, None, None]
    assert g(ctypes.byref(c), *good, 0, None) == BAD  # no workspace
    good[14] = 64
    for at, bad in ((0, None), (8, None), (9, None), (10, None), (11, None), (12, None), (13, 64), (9, 68)):
        args = list(good)
        args[at] = bad
        assert g(ctypes.byref(c), *args, 1 << 30, None) == BAD, (at, bad)


def test_bias_and_dropout_refuse():
    borders = (ctypes.c_int * 3)(1, 2, 2)

    def bias(**change):
        c = _lib.rg_relative_bias_config(3, 4, 0, 2, 3, 0, 1, borders)
        for n, v in change.items():
            setattr(c, n, v)
        return _lib.lib.rg_relative_bias_fp32(ctypes.byref(c), None, None, None)

    for change in (dict(Tq=-1), dict(Tk=2 ** 23), dict(H=0), dict(count=0), dict(count=513), dict(borders=None),
                   dict(borders=(ctypes.c_int * 3)(0, 1, 2)), dict(borders=(ctypes.c_int * 3)(3, 2, 4)), dict()):
        assert bias(**change) == BAD, change
    assert bias(Tq=0) == 0
    f = _lib.lib.rg_dropout_fp32
    for args in ((64, 64, 4, 1.0, 0, None, None), (64, 64, 4, -1.0, 0, None, None), (None, 64, 4, 0.5, 0, None, None),
                 (64, 66, 4, 0.5, 0, None, None), (64, 64, 4, 0.5, 0, 68, None), (64, 64, 4, 0.5, 0, None, 68)):
        assert f(*args, None) == BAD, args
    assert f(None, None, 0, 0.5, 0, None, None, None) == 0
