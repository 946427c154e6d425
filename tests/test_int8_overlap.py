"""add_rmsnorm writes h_out row by row while others are still read: it may be h, or y of its type, place for place, and
nothing else of theirs or the weight's (without a GPU: refused before a device is touched)."""

import ctypes

import pytest

from opac1ty_b200 import _lib

F16, F32 = _lib.OPC_F16, _lib.OPC_F32
H, Y, W = 1 << 20, 1 << 21, 1 << 22  # aligned addresses that nothing reads
N, LD = 48, 128


def norm(h_out, ldho=N, h=H, ldh=N, y=Y, ldy=N, y_type=F16, w=W, rows=4):
    """Whether the call is refused for its memory.  (eps is refused after that.)"""
    c = _lib.I8Rows(rows, N, N, 1 << 24, 1 << 25)
    rc = _lib.load().opc_i8_add_rmsnorm(h, ldh, F32, y, ldy, y_type, w, F16, 0.0, h_out, ldho, ctypes.byref(c), None, 0, 0, None)
    assert rc == _lib.OPC_ERR_INVALID and ("overlap" in _lib.last_error()) != ("eps" in _lib.last_error())
    return "overlap" in _lib.last_error()


@pytest.mark.parametrize("kw", [
    dict(h_out=H), dict(h_out=None), dict(h_out=1 << 23), dict(h_out=Y, y_type=F32), dict(h_out=H, y=H, y_type=F32),
    dict(h_out=H + 4 * 4 * N),                                              # right behind h
    dict(h_out=H + 4 * N, ldho=LD, ldh=LD),                                 # beside it in rows of 128
    dict(h_out=H + 4 * (LD - N), ldho=LD, ldh=LD), dict(h_out=H - 4 * N, ldho=LD, ldh=LD),
    dict(h_out=H, ldho=LD, rows=1), dict(h_out=H, y=None), dict(h_out=H, w=None),
    dict(h_out=H, ldho=LD, ldh=LD, w=H + 4 * N),                            # the weight between two rows
])
def test_taken(kw):
    assert not norm(**kw)


@pytest.mark.parametrize("kw", [
    dict(h_out=H + 4), dict(h_out=H + 4 * N), dict(h_out=H - 4 * N), dict(h_out=H + 4 * 4 * N - 4),
    dict(h_out=H, ldho=LD), dict(h_out=H, ldh=LD), dict(h_out=H + 4 * (N - 1), ldho=LD, ldh=LD),
    dict(h_out=H + 4 * (LD - N + 1), ldho=LD, ldh=LD), dict(h_out=H + 4, rows=1),
    dict(h_out=Y), dict(h_out=Y, y_type=F32, ldho=LD), dict(h_out=Y + 8, y_type=F32), dict(h_out=Y + 2 * 4 * N - 4),
    dict(h_out=W), dict(h_out=W + 2 * N - 4), dict(h_out=W - 4 * 3 * N), dict(h_out=H, w=H), dict(h_out=H, w=H + 4 * N),
    dict(h_out=H, ldho=LD, ldh=LD, w=H + 4 * LD - 2),
])
def test_refused(kw):
    assert norm(**kw)
