"""Orthogonalised updates: a workspace in the memory of the matrices is refused (in front of any launch: no GPU needed)."""
import pytest

from encodermap_amd import _lib

P = 1 << 20    # addresses that nothing reads
G, W, M, OUT = P, 2 * P, 3 * P, 4 * P
MATS = (_lib.Matrix * 2)()
for e, (offset, rows, cols) in zip(MATS, [(10, 8, 4), (50, 3, 3)]):     # elements 10 .. 59
    e.offset, e.rows, e.cols, e.ld, e.scale = offset, rows, cols, cols, 1.0
NEED = _lib.load().emx_orthogonalize_ws_bytes(MATS, 2)


def orthogonalize(ws, g=G, out=OUT):
    return _lib.load().emx_orthogonalize(MATS, 2, g, out, 0, 5, 1e-7, ws, NEED, None)


def step(ws, slices=1, stride=0):
    return _lib.load().emx_muon_step(MATS, 2, W, G, slices, stride, M, 0.1, 0.9, 1, 0.0, 5, 1e-7, ws, NEED, None)


@pytest.mark.parametrize("ws", [G, G + 128, G + 48, G - NEED + 48, OUT + 224, OUT - 16])
def test_orthogonalize(ws):
    assert NEED % 16 == 0
    assert orthogonalize(ws) == -1 and b"workspace" in _lib.load().emx_last_error()


def test_in_place():
    assert orthogonalize(G + 64, g=G, out=G) == -1 and b"workspace" in _lib.load().emx_last_error()


@pytest.mark.parametrize("ws", [G, W + 32, W + 224, M, M - NEED + 48])
def test_step(ws):
    assert step(ws) == -1 and b"workspace" in _lib.load().emx_last_error()


def test_a_slice_of_the_gradient():
    """the third of three slices, 4096 elements apart, ends at element 2 x 4096 + 59"""
    far = G + 4 * (2 * 4096 + 58) // 16 * 16
    assert step(far, slices=3, stride=4096) == -1 and b"workspace" in _lib.load().emx_last_error()
