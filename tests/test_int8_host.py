"""The 8-bit products' C entry points without a GPU: every refusal comes before a device is touched."""

import ctypes

import pytest

from opac1ty_b200 import _lib

P = 1 << 12  # an aligned address that nothing reads


def rows(rows=4, n=48, ld=48, codes=P, scales=P):
    return _lib.I8Rows(rows, n, ld, codes, scales)


def quantize(out, x=P, ldx=48, dtype=_lib.OPC_F16, values=None, ldv=0, v_dtype=0):
    return _lib.load().opc_i8_quantize(x, ldx, dtype, ctypes.byref(out) if out is not None else None, values, ldv, v_dtype, None)


def norm(out, h=P, ldh=48, ht=_lib.OPC_F32, y=P, ldy=48, yt=_lib.OPC_F16, w=P, wt=_lib.OPC_F16, eps=1e-5, ho=P, ldho=48):
    return _lib.load().opc_i8_add_rmsnorm(h, ldh, ht, y, ldy, yt, w, wt, eps, ho, ldho, ctypes.byref(out), None, 0, 0, None)


def gemm(x, w, bias=None, bt=0, y=P, ldy=64, yt=_lib.OPC_F16):
    return _lib.load().opc_i8_gemm(ctypes.byref(x), ctypes.byref(w), bias, bt, y, ldy, yt, None)


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(rows=2**31 - 4095), dict(n=0), dict(n=131072), dict(ld=47), dict(ld=32), dict(ld=56),
                                dict(codes=None), dict(codes=P + 8), dict(scales=None), dict(scales=P + 2)])
def test_rows_of_codes_are_checked(kw):
    if kw.get("n") == 131072:
        kw["ld"] = 131072
    bad = rows(**kw)
    for rc in (quantize(bad), norm(bad), gemm(bad, rows(rows=64)), gemm(rows(), bad),
               _lib.load().opc_i8_silu_mul(P, 48, P, 48, _lib.OPC_F16, ctypes.byref(bad), None, 0, 0, None)):
        assert rc == _lib.OPC_ERR_INVALID and "opc_i8_" in _lib.last_error()
    assert quantize(None) == _lib.OPC_ERR_INVALID


@pytest.mark.parametrize("kw,code", [
    (dict(x=None), _lib.OPC_ERR_INVALID), (dict(x=P + 1), _lib.OPC_ERR_INVALID), (dict(ldx=47), _lib.OPC_ERR_INVALID),
    (dict(dtype=3), _lib.OPC_ERR_UNSUPPORTED), (dict(dtype=_lib.OPC_F32, x=P + 2), _lib.OPC_ERR_INVALID),
    (dict(values=P, ldv=47), _lib.OPC_ERR_INVALID), (dict(values=P, ldv=48, v_dtype=9), _lib.OPC_ERR_UNSUPPORTED),
    (dict(values=P + 1, ldv=48), _lib.OPC_ERR_INVALID)])
def test_quantize_refuses(kw, code):
    assert quantize(rows(), **kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(h=None), _lib.OPC_ERR_INVALID), (dict(ldh=4), _lib.OPC_ERR_INVALID), (dict(ldy=4), _lib.OPC_ERR_INVALID),
    (dict(yt=5), _lib.OPC_ERR_UNSUPPORTED), (dict(ht=_lib.OPC_F16, yt=_lib.OPC_BF16), _lib.OPC_ERR_UNSUPPORTED),
    (dict(ht=_lib.OPC_BF16, yt=_lib.OPC_F32), _lib.OPC_ERR_UNSUPPORTED), (dict(w=P + 1), _lib.OPC_ERR_INVALID),
    (dict(wt=7), _lib.OPC_ERR_UNSUPPORTED), (dict(ldho=40), _lib.OPC_ERR_INVALID), (dict(ho=P + 2), _lib.OPC_ERR_INVALID),
    (dict(eps=0.0), _lib.OPC_ERR_INVALID), (dict(eps=1e-13), _lib.OPC_ERR_INVALID), (dict(eps=float("nan")), _lib.OPC_ERR_INVALID),
    (dict(eps=float("inf")), _lib.OPC_ERR_INVALID)])
def test_norm_refuses(kw, code):
    assert norm(rows(), **kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(y=None), _lib.OPC_ERR_INVALID), (dict(ldy=63), _lib.OPC_ERR_INVALID), (dict(yt=3), _lib.OPC_ERR_UNSUPPORTED),
    (dict(bias=P, bt=4), _lib.OPC_ERR_UNSUPPORTED), (dict(bias=P + 1), _lib.OPC_ERR_INVALID)])
def test_gemm_refuses(kw, code):
    assert gemm(rows(), rows(rows=64), **kw) == code


def test_gemm_refuses_unlike_widths_and_no_channels():
    assert gemm(rows(n=40), rows(rows=64)) == _lib.OPC_ERR_INVALID and "rows of 40" in _lib.last_error()
    assert gemm(rows(), rows(rows=0)) == _lib.OPC_ERR_INVALID and "no rows" in _lib.last_error()


def test_no_rows_are_nothing_to_do():
    none = rows(rows=0, codes=None, scales=None)
    assert quantize(none, x=None) == norm(none, h=None) == gemm(none, rows(rows=64), y=None) == _lib.OPC_OK
