"""Argument checks of the sorted-token entry points: every refusal is made on the host, before any
launch, so none of them needs a GPU (the addresses are never read)."""

import pytest

from vybforge_b200 import _lib

A = 1 << 20  # a well-aligned address


def permute(lib, idx=A, T=4, k=2, E=16, x=A, dt=0, H=64, xs=A, counts=A, offsets=A, perm=A, pos=A):
    return lib.vfmoe_permute(idx, T, k, E, x, dt, H, xs, counts, offsets, perm, pos, 0)


@pytest.mark.parametrize("kw", [dict(idx=0), dict(T=-1), dict(k=0), dict(k=33), dict(E=0), dict(E=1025), dict(dt=3),
                                dict(dt=-1), dict(H=0), dict(xs=0), dict(counts=0), dict(offsets=0), dict(perm=0),
                                dict(pos=0), dict(x=A + 2), dict(xs=A + 1, dt=1), dict(pos=A + 2), dict(T=1 << 40),
                                dict(T=1 << 30, k=2)])
def test_permute_refuses(built_lib, kw):
    assert permute(built_lib, **kw) == _lib.ERR_INVALID
    assert "vfmoe_permute" in _lib.last_error()


@pytest.mark.parametrize("kw", [dict(y=0), dict(dt=5), dict(pos=0), dict(T=-2), dict(k=0), dict(k=40), dict(H=0),
                                dict(out=0), dict(odt=9), dict(y=A + 2), dict(out=A + 2), dict(pos=A + 1)])
def test_permute_backward_and_combine_refuse(built_lib, kw):
    a = dict(y=A, dt=0, pos=A, T=4, k=2, H=64, out=A, odt=0)
    a.update(kw)
    assert built_lib.vfmoe_permute_backward(a["y"], a["dt"], a["pos"], a["T"], a["k"], a["H"], a["out"], a["odt"],
                                            0) == _lib.ERR_INVALID
    assert built_lib.vfmoe_combine(a["y"], a["dt"], a["pos"], 0, a["T"], a["k"], a["H"], 0, a["out"], a["odt"],
                                   0) == _lib.ERR_INVALID


@pytest.mark.parametrize("kw", [dict(dout=0), dict(y=0), dict(dy=0, dw=0), dict(pos=0), dict(gt=4), dict(yt=-2),
                                dict(k=33), dict(H=-1), dict(dy=A + 1), dict(dw=A + 2), dict(dout=A + 2)])
def test_combine_backward_refuses(built_lib, kw):
    a = dict(dout=A, gt=0, y=A, yt=0, pos=A, w=0, T=4, k=2, H=64, dy=A, dw=A)
    a.update(kw)
    assert built_lib.vfmoe_combine_backward(a["dout"], a["gt"], a["y"], a["yt"], a["pos"], a["w"], a["T"], a["k"],
                                            a["H"], a["dy"], a["dw"], 0) == _lib.ERR_INVALID


def test_nothing_to_do_is_no_error(built_lib):
    assert built_lib.vfmoe_combine(0, 0, 0, 0, 0, 2, 64, 0, 0, 0, 0) == _lib.OK
    assert built_lib.vfmoe_combine_backward(0, 0, 0, 0, 0, 0, 0, 2, 64, 0, 0, 0) == _lib.OK
    assert built_lib.vfmoe_permute_backward(0, 0, 0, 0, 2, 64, 0, 0, 0) == _lib.OK


@pytest.mark.parametrize("kw", [dict(T=1 << 31), dict(H=1 << 31), dict(k=33), dict(T=1 << 27, k=64)])
def test_combine_refuses_what_passes_its_indices(built_lib, kw):
    a = dict(T=4, k=2, H=64)
    a.update(kw)
    assert built_lib.vfmoe_combine(A, 0, A, 0, a["T"], a["k"], a["H"], 0, A, 0, 0) == _lib.ERR_INVALID
