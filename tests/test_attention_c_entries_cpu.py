"""The C entries of rotary positions and attention over another sequence refuse what their kernels could not read or write, before anything is launched."""
import ctypes
from ctypes import POINTER, Structure, byref, c_float, c_int, c_longlong, c_void_p

import pytest

from flodl_b200 import _ext


class Rotary(Structure):
    _fields_ = [("x", c_void_p * 3), ("dy", c_void_p * 3), ("y", c_void_p * 3), ("x_strides", c_longlong * 9), ("dy_strides", c_longlong * 9), ("y_strides", c_longlong * 9),
                ("heads", c_int * 3), ("B", c_int), ("S", c_int), ("D", c_int), ("rot", c_int), ("dtype", c_int), ("interleaved", c_int), ("norm", c_int), ("backward", c_int),
                ("amplitude", c_float), ("eps", c_float), ("freqs", c_void_p), ("positions", c_void_p), ("pos_strides", c_longlong * 2), ("offset", c_longlong),
                ("weight", c_void_p * 2), ("partial", c_void_p), ("dw", c_void_p * 2)]


class Cross(Structure):
    _fields_ = [(n, c_void_p) for n in ("q", "k", "v", "d_o", "o", "dq", "dk", "dv")] + \
               [(n + "_strides", c_longlong * 3) for n in ("q", "k", "v", "o", "do", "dq", "dk")] + \
               [(n, c_int) for n in ("B", "H", "Hk", "Sq", "Sk", "D")] + \
               [("mask", c_void_p), ("mask_stride", c_longlong), ("mask_bool", c_int), ("scale", c_float), ("stats", c_void_p), ("mask_info", c_void_p), ("workspace", c_void_p),
                ("status", c_void_p)]


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(_ext.require().__file__)
    for name, kind in (("fb_rotary", Rotary), ("fb_cross_attn_fwd", Cross), ("fb_cross_attn_bwd", Cross)):
        getattr(lib, name).argtypes = [POINTER(kind), c_void_p]
    lib.fb_cross_workspace.argtypes = [POINTER(Cross), c_int]
    lib.fb_cross_mask_info.argtypes = [POINTER(Cross)]
    lib.fb_cross_workspace.restype = lib.fb_cross_mask_info.restype = c_longlong
    return lib


AT = 1 << 20            # an address that nothing reads


def rotary(**kw):
    a = Rotary(B=2, S=3, D=64, rot=64, dtype=6, norm=1, backward=1, amplitude=1.0, eps=1e-6, freqs=AT, positions=AT, partial=AT)
    for i in range(3):
        a.x[i] = a.dy[i] = a.y[i] = AT
        a.heads[i] = 4
    a.weight[0] = a.weight[1] = a.dw[0] = a.dw[1] = AT
    for n, v in kw.items():
        if isinstance(v, tuple):
            getattr(a, n)[v[0]] = v[1]
        else:
            setattr(a, n, v)
    return a


def cross(**kw):
    a = Cross(B=2, H=4, Hk=2, Sq=5, Sk=70, D=64, scale=0.125, **{n: AT for n in ("q", "k", "v", "d_o", "o", "dq", "dk", "dv", "mask", "stats", "mask_info", "workspace", "status")})
    for n in ("q", "k", "v", "o", "do", "dq", "dk"):
        getattr(a, n + "_strides")[:] = [70 * 4 * 64, 4 * 64, 64]
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def test_null_arguments(lib):
    assert lib.fb_rotary(None, None) == lib.fb_cross_attn_fwd(None, None) == lib.fb_cross_attn_bwd(None, None) == -3
    assert lib.fb_cross_workspace(None, 1) == lib.fb_cross_mask_info(None) == -3


@pytest.mark.parametrize("kw", [dict(x=(0, AT + 2)), dict(dy=(1, AT + 1)), dict(y=(2, AT + 3)), dict(freqs=AT + 4), dict(positions=AT + 4), dict(partial=AT + 2), dict(weight=(1, AT + 2)),
                                dict(dw=(0, AT + 1)), dict(freqs=None), dict(partial=None), dict(x=(0, None)), dict(dy=(2, None)), dict(y=(1, None))], ids=str)
def test_rotary(lib, kw):
    assert lib.fb_rotary(byref(rotary(**kw)), None) == -3


@pytest.mark.parametrize("kw", [dict(q=AT + 8), dict(k=AT + 2), dict(v=None), dict(o=AT + 8), dict(mask=AT + 2), dict(mask_info=None), dict(mask_info=AT + 1), dict(stats=AT + 2),
                                dict(workspace=AT + 8), dict(status=AT + 2)], ids=str)
def test_cross(lib, kw):
    assert lib.fb_cross_attn_fwd(byref(cross(**kw)), None) == -3
    assert lib.fb_cross_attn_bwd(byref(cross(**kw)), None) == -3


@pytest.mark.parametrize("kw", [dict(stats=None), dict(workspace=None), dict(dq=None, dk=None, dv=None), dict(dk=None), dict(dv=None), dict(dq=AT + 8), dict(dv=AT + 4), dict(d_o=None)], ids=str)
def test_cross_backward(lib, kw):
    assert lib.fb_cross_attn_bwd(byref(cross(**kw)), None) == -3


@pytest.mark.parametrize("kw", [dict(D=80), dict(Hk=3), dict(B=0), dict(Sq=0), dict(Sk=0), dict(H=0), dict(Hk=0)], ids=str)
def test_sizes(lib, kw):
    assert lib.fb_cross_attn_fwd(byref(cross(**kw)), None) == lib.fb_cross_attn_bwd(byref(cross(**kw)), None) == -4
    assert lib.fb_cross_mask_info(byref(cross(**kw))) == -4


def test_what_a_mask_comes_to(lib):
    """Live blocks and a base of each batch row, its list of blocks; of many batch rows where each is among the tiles."""
    assert lib.fb_cross_mask_info(byref(cross())) == 2 * (2 + 1) and lib.fb_cross_mask_info(byref(cross(mask=None))) == 0
    assert lib.fb_cross_mask_info(byref(cross(B=65, Sk=300))) == 65 * (2 + 3) + 2 * 66
