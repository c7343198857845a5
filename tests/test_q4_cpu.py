"""Argument checks of the 4-bit entry points: refused on the host before any launch, without a GPU (the
addresses are never read)."""

import ctypes as C

import pytest

from vybforge_b200 import _lib

A = 1 << 20


def mat(**kw):
    d = dict(n=32, k=128, group=32, n_mats=1, scale_dtype=_lib.DT_BF16, data=A, scales=A, zeros=A)
    d.update(kw)
    return _lib.Q4Desc(**d)


BAD_MATS = [dict(n=0), dict(n=24), dict(k=0), dict(k=96, group=64), dict(group=16), dict(group=256, k=512), dict(n_mats=0),
            dict(n_mats=1025), dict(scale_dtype=_lib.DT_F32), dict(data=0), dict(scales=0), dict(data=A + 8),
            dict(scales=A + 2), dict(zeros=A + 1)]


def matvec(lib, w=None, up=None, limit=10.0, x=A, xd=0, xr=4, rm=0, off=0, rows=4, y=A, yd=0):
    w = mat() if w is None else w
    return lib.vfmoe_q4_matvec(C.byref(w), None if up is None else C.byref(up), limit, x, xd, xr, rm, off, rows, y, yd, 0)


def test_descriptor_is_a_block_of_8_byte_words():
    assert C.sizeof(_lib.Q4Desc) == 8 * 8


@pytest.mark.parametrize("kw", BAD_MATS)
def test_bad_matrices(built_lib, kw):
    assert matvec(built_lib, mat(**kw)) == _lib.ERR_INVALID
    assert "bad 4-bit matrix" in _lib.last_error()
    assert matvec(built_lib, up=mat(**kw)) == _lib.ERR_INVALID
    assert built_lib.vfmoe_q4_quantize(A, 0, C.byref(mat(**kw)), 0) == _lib.ERR_INVALID
    assert built_lib.vfmoe_q4_dequant(C.byref(mat(**kw)), A, 0, 0) == _lib.ERR_INVALID


@pytest.mark.parametrize("kw", [dict(n=48), dict(k=256), dict(group=64), dict(n_mats=2), dict(scale_dtype=_lib.DT_F16),
                                dict(zeros=0)])
def test_up_must_match(built_lib, kw):
    assert matvec(built_lib, up=mat(**kw)) == _lib.ERR_INVALID
    assert "up must have" in _lib.last_error()


@pytest.mark.parametrize("kw", [dict(x=0), dict(y=0), dict(xd=3), dict(yd=-1), dict(rows=-1), dict(rows=1 << 31), dict(xr=3),
                                dict(xr=-1), dict(x=A + 4), dict(y=A + 8), dict(rm=A + 2), dict(off=A + 1),
                                dict(w=mat(n_mats=2))])
def test_bad_arguments(built_lib, kw):
    assert matvec(built_lib, **kw) == _lib.ERR_INVALID


def test_null_and_empty(built_lib):
    assert built_lib.vfmoe_q4_matvec(None, None, 10.0, A, 0, 4, 0, 0, 4, A, 0, 0) == _lib.ERR_INVALID
    assert matvec(built_lib, rows=0, x=0, y=0, xr=0) == _lib.OK
    for limit in (0.0, -1.0, float("nan")):
        assert matvec(built_lib, up=mat(), limit=limit) == _lib.ERR_INVALID
    assert built_lib.vfmoe_q4_quantize(0, 0, C.byref(mat()), 0) == _lib.ERR_INVALID
    assert built_lib.vfmoe_q4_quantize(A, 4, C.byref(mat()), 0) == _lib.ERR_INVALID
    assert built_lib.vfmoe_q4_dequant(C.byref(mat()), A + 2, 0, 0) == _lib.ERR_INVALID


def test_dequant_checks_where_the_matrix_lies():
    """A matrix that is not on the current device is refused before its addresses reach a kernel of that device."""
    import torch

    from vybforge_b200 import moe
    m = object.__new__(moe.Q4Matrix)                       # as if made while another device was current
    m.codes, m.scales, m.zeros = torch.zeros(32, 64, dtype=torch.uint8), torch.zeros(4, 32).half(), None
    m.N, m.K, m.group, m.n_mats = 32, 128, 32, 1
    m.desc = mat(zeros=0, scale_dtype=_lib.DT_F16)
    with pytest.raises(_lib.VfmoeError) as e:
        moe.q4_dequant(m)
    assert e.value.code == _lib.ERR_INVALID and "current" in str(e.value)
