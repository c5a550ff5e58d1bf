"""Layer norm on the CPU side: what emx_layernorm_* refuses (before any launch: no GPU needed), the scratch it asks for, the binding's checks."""
import ctypes as C

import pytest
import torch

from encodermap_amd import _lib

P = 1 << 20    # an address that nothing reads: every call here is refused in front of its launch


def fwd(x=P, dtype=0, n=4, D=8, ldx=8, eps=1e-3, y=2 * P, ldy=8):
    return _lib.load().emx_layernorm_fwd(x, dtype, n, D, ldx, None, None, eps, y, ldy, None, None, None)


def bwd(dy=P, ld_dy=8, x=2 * P, ldx=8, dtype=0, n=4, D=8, mean=3 * P, rstd=3 * P, dx=4 * P, ld_dx=8, dgamma=5 * P, dbeta=5 * P, ws=6 * P, ws_floats=None):
    need = _lib.layernorm_ws_floats(max(n, 0), max(D, 1)) if ws_floats is None else ws_floats
    return _lib.load().emx_layernorm_bwd(dy, ld_dy, x, ldx, dtype, n, D, None, mean, rstd, dx, ld_dx, dgamma, dbeta, ws, need, None)


@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(dtype=-1), dict(n=-1), dict(D=0), dict(D=-4), dict(D=(1 << 28) + 1), dict(eps=-1e-6), dict(eps=float("nan")), dict(x=None),
    dict(y=None), dict(ldx=-8), dict(ldy=7), dict(ldy=0),
    dict(y=P + 4),               # shifted rows of the same memory
    dict(y=P, ldx=8, ldy=16),    # the same start with another stride
    dict(y=P + 4 * 31),          # the first row of one is the end of the other
    dict(x=P + 2), dict(y=2 * P + 1),                     # not on an element boundary
    dict(n=1 << 40, ldx=1 << 30), dict(n=1 << 40, ldy=1 << 30),
])
def test_forward_refuses(bad):
    assert fwd(**bad) == -1
    assert b"emx_layernorm_fwd" in _lib.load().emx_last_error()


@pytest.mark.parametrize("bad", [
    dict(dtype=9), dict(n=-1), dict(D=0), dict(dy=None), dict(x=None), dict(mean=None), dict(rstd=None), dict(ldx=-1), dict(ld_dy=-1), dict(ld_dx=7),
    dict(dx=P + 4), dict(dx=2 * P - 4), dict(dx=P, ld_dx=16), dict(dy=P + 1), dict(x=2 * P + 2), dict(dx=4 * P + 3), dict(n=1 << 40, ldx=1 << 30, ws_floats=1 << 40),
])
def test_backward_refuses(bad):
    assert bwd(**bad) == -1
    assert b"emx_layernorm_bwd" in _lib.load().emx_last_error()


def test_backward_refuses_a_short_workspace():
    need = _lib.layernorm_ws_floats(4, 8)
    assert need >= 16
    assert bwd(ws_floats=need - 1) == -4 and bwd(ws=None) == -4


def test_no_rows_is_no_launch():
    before = _lib.load().emx_launch_count()
    assert fwd(x=None, n=0, y=None) == 0
    assert bwd(dy=None, x=None, n=0, mean=None, rstd=None, dx=None, dgamma=None, dbeta=None, ws=None) == 0
    assert _lib.load().emx_launch_count() == before


@pytest.mark.parametrize("n,D", [(0, 8), (1, 1), (1, 1 << 20), (16, 128), (17, 128), (4096, 128), (1000000, 128), (65536, 1024), (1 << 40, 8), (100, 1 << 28)])
def test_workspace_is_two_sums_per_column_and_part(n, D):
    floats = _lib.layernorm_ws_floats(n, D)
    assert floats % (2 * D) == 0
    assert (floats == 0) == (n == 0)
    assert floats // (2 * D) <= max(1, (n + 7) // 8)     # (eight rows and more to a part)
    assert floats <= max(64 * D, 8 << 20)


def test_the_binding_refuses_what_is_no_row_block_of_a_gpu():
    x = torch.zeros(4, 8)
    with pytest.raises(_lib.EmxError, match="GPU"):
        _lib.layernorm_fwd(x, None, None, 1e-3, torch.zeros(4, 8))
    with pytest.raises(_lib.EmxError, match="float64"):
        _lib.layernorm_fwd(x.double(), None, None, 1e-3, x.double())
    assert C.sizeof(C.c_void_p) == 8
