"""Orthogonalised updates on the CPU side: what emx_orthogonalize / emx_muon_step refuse (before any launch: no GPU needed) and the scratch they ask for."""
import ctypes as C

import pytest
import torch

from encodermap_amd import _lib
from encodermap_amd.layout import build_layout

P = 1 << 20    # an address that nothing reads: every call here is refused in front of its launch


def table(*mats):
    t = (_lib.Matrix * max(len(mats), 1))()
    for e, m in zip(t, mats):
        e.offset, e.rows, e.cols, e.ld, e.scale = (tuple(m) + (m[2], 1.0))[:5] if len(m) == 3 else (tuple(m) + (1.0,))[:5]
    return t, len(mats)


def need(*mats):
    return _lib.load().emx_orthogonalize_ws_bytes(*table(*mats))


def ortho(mats, g=P, out=2 * P, dtype=0, steps=5, eps=1e-7, ws=3 * P, ws_bytes=None):
    t, n = table(*mats)
    return _lib.load().emx_orthogonalize(t, n, g, out, dtype, steps, eps, ws, need(*mats) if ws_bytes is None else ws_bytes, None)


def muon(mats, w=P, g=2 * P, slices=1, stride=0, m=3 * P, lr=0.1, beta=0.9, decay=0.0, steps=5, eps=1e-7, ws=4 * P, ws_bytes=None):
    t, n = table(*mats)
    return _lib.load().emx_muon_step(t, n, w, g, slices, stride, m, lr, beta, 1, decay, steps, eps, ws, need(*mats) if ws_bytes is None else ws_bytes, None)


ONE = [(0, 8, 4)]


@pytest.mark.parametrize("mats,code", [
    ([(-1, 8, 4)], -1), ([(0, -8, 4)], -1), ([(0, 8, -4)], -1), ([(0, 8, 4, 3)], -1), ([(0, 8, 4, -4)], -1), ([(0, 8, 4, 1 << 41)], -1),
    ([(0, 8, 40000)], -2), ([(0, 40000, 8)], -2),
    ([(0, 8, 4), (0, 8, 4)], -1),                    # the same matrix twice
    ([(0, 8, 4), (31, 8, 4)], -1),                   # the last element of one is the first of the other
    ([(0, 8, 4, 10), (3, 8, 4, 10)], -1),            # column blocks that share a column
    ([(0, 8, 4, 10), (8, 8, 4, 10)], -1),            # ... that run over the row's end into the next row's first columns
    ([(0, 8, 4, 10), (5, 8, 4, 11)], -1),            # rows of two lengths between one another
    ([(100, 2, 2), (0, 60, 4, 4), (96, 1, 8)], -1), ([((1 << 50) + 1, 2, 2)], -1),
])
def test_matrices_that_are_refused(mats, code):
    assert need(*mats) == 0
    assert ortho(mats, ws_bytes=1 << 40) == code and muon(mats, ws_bytes=1 << 40) == code
    assert b"matri" in _lib.load().emx_last_error()


@pytest.mark.parametrize("mats", [
    [], [(0, 0, 4)], [(0, 4, 0)], [(0, 1, 5, 0)], [(0, 8, 4), (32, 8, 4)], [(32, 8, 4), (0, 8, 4)], [(0, 8, 4, 10), (4, 8, 6, 10)],
    [(0, 8, 4, 10), (4, 1, 6)], [(7, 32768, 1)], [(0, 8, 4), (0, 0, 9)],
])
def test_matrices_that_are_taken(mats):
    assert need(*mats) >= 16


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(steps=0), dict(steps=65), dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")),
                                 dict(g=None), dict(out=None), dict(g=P + 2), dict(out=2 * P + 1), dict(out=P + 4), dict(out=P - 4 * 31)])
def test_orthogonalize_refuses(bad):
    assert ortho(ONE, **bad) == -1
    assert b"emx_orthogonalize" in _lib.load().emx_last_error()


@pytest.mark.parametrize("bad", [dict(slices=0), dict(slices=2, stride=-1), dict(lr=float("nan")), dict(lr=float("inf")), dict(beta=1.0), dict(beta=-0.1),
                                 dict(beta=float("nan")), dict(decay=float("nan")), dict(steps=0), dict(steps=65), dict(eps=0.0), dict(w=None), dict(g=None),
                                 dict(m=None), dict(w=2 * P), dict(m=P), dict(m=2 * P), dict(w=P + 2), dict(m=P + 4), dict(w=2 * P + 4 * 31),
                                 dict(g=P - 4 * 99, slices=2, stride=100), dict(slices=3, stride=1 << 60)])
def test_muon_refuses(bad):
    assert muon(ONE, **bad) == -1
    assert b"emx_muon_step" in _lib.load().emx_last_error()


def test_muon_refuses_a_scale_that_is_no_number():
    assert muon([(0, 8, 4, 4, float("nan"))]) == -1 and muon([(0, 8, 4, 4, float("inf"))]) == -1


def test_the_workspace_is_checked():
    n = need(*ONE)
    for call in (ortho, muon):
        assert call(ONE, ws_bytes=n - 1) == -4 and call(ONE, ws=None) == -4 and call(ONE, ws=4 * P + 8) == -4


def test_nothing_to_do_is_no_launch():
    before = _lib.load().emx_launch_count()
    assert ortho([], g=None, out=None, ws=None) == 0 and muon([(0, 0, 3)], w=None, g=None, m=None, ws=None) == 0
    assert _lib.load().emx_launch_count() == before


def test_the_workspace_serves_groups_in_turn():
    """more matrices than one launch takes: the groups use the same scratch, one after the other"""
    many = [(16 * i, 4, 4) for i in range(200)]
    assert need(*many) == need(*many[:64]) > need(*many[:10])


def test_plan_of_a_layout():
    lay = build_layout([128, 128, 2], ["", "tanh", "tanh", ""], 128)
    plan = _lib.MatrixPlan.of_layers(lay.layers, device="cpu")
    assert plan.n == 6 and plan.end == lay.layers[-1].w_off + 128 * 128
    assert [plan.mats[i].scale for i in range(6)] == [1.0, 1.0, 1.0, 8.0, 1.0, 1.0]
    with pytest.raises(_lib.EmxError, match="GPU"):
        _lib.orthogonalize(plan, torch.zeros(lay.n_params), torch.zeros(lay.n_params))
    with pytest.raises(_lib.EmxError, match="overlap"):
        _lib.MatrixPlan([(0, 4, 4, 4, 1.0), (15, 4, 4, 4, 1.0)], device="cpu")
    for bad in ((0, 2 ** 32 + 4, 4, 4, 1.0), (0, 4, 2 ** 32 + 4, 4, 1.0), (-1, 4, 4, 4, 1.0), (0, 4, 4, 2 ** 64 + 4, 1.0)):
        with pytest.raises(_lib.EmxError):
            _lib.MatrixPlan([bad], device="cpu")
    assert C.sizeof(_lib.Matrix) == 32
