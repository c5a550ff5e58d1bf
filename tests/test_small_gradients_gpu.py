"""Gradients that are small beside the eps of the orthogonalisation: X_0 = G / (|G|_F + eps) is small then, and its result is as exact, relative to ITS size, as that
of any other -- at the default eps, in every kernel that a matrix' size leads to.

Tolerance: that of test_muon_gpu.py with the size of X_0 in it.  2^-20 of |X_k|_F per step, times the 3.4445^(steps - k) that the steps behind it make of it, where
|X_k|_F <= min(3.4445^k |X_0|_F, 1.2024 sqrt(M)).  As long as the result is small itself, it is 3.4445^steps X_0 and this is 6 x 2^-20 of it.  Results of 16 bits
are rounded once more."""
import math

import pytest
import torch

from tests import test_muon_gpu as om

pytestmark = pytest.mark.gpu

EPS = 1e-7
NORMS = [1e-5, 1e-7, 3e-8, 1e-9, 1e-12, 1e-14, 1e-16, 1e-20, 1e-30]


@pytest.fixture(scope="module")
def lib():
    from encodermap_amd import _lib

    _lib.require_gpu()
    return _lib


def allowed(shape, start, steps):
    side = min(shape)
    return om.STEP * sum(om.ABC[0] ** (steps - k) * min(om.ABC[0] ** k * start, 1.2024 * math.sqrt(side)) for k in range(steps + 1))


def small(rows, cols, norm, seed):
    g = om.gradient(rows, cols, seed)
    return g * (norm / g.double().norm().item())


def check(got, g, steps, what):
    want = om.iterate(g.double(), steps, EPS)
    n = g.double().norm().item()
    limit = allowed(g.shape, n / (n + EPS), steps)
    assert torch.isfinite(got).all(), what
    err = (got.double() - want).abs()
    if got.dtype != torch.float32:
        err = (err - torch.finfo(got.dtype).eps / 2 * 1.01 * want.abs()).clamp_min(0)
    assert err.norm().item() <= limit, f"{what}: {err.norm().item() / want.norm().item():.3g} of the result off, {limit / want.norm().item():.3g} allowed"


def run(lib, shapes, norms, kind="f32", steps=5):
    entries, n = om.lay_out(shapes)
    flat = torch.zeros(n, device="cuda").to(om.TYPES[kind])
    for i, (v, norm) in enumerate(zip(om.views(flat, entries), norms)):
        v.copy_(small(*v.shape, norm, i))
    out = torch.zeros_like(flat)
    lib.orthogonalize(lib.MatrixPlan(entries), flat, out, steps=steps)
    for shape, norm, g, o in zip(shapes, norms, om.views(flat, entries), om.views(out, entries)):
        check(o, g, steps, f"{shape}, norm {norm:g}, {steps} steps, {kind}")


# sixteen rows and fewer; up to 128, of one and of several strips; 64 x 64 tiles, with the first product in parts too; larger ones
SHAPES = [(2, 128), (300, 9), (20, 30), (128, 128), (64, 97), (100, 400), (4100, 128), (150, 130), (333, 999), (9000, 200), (1100, 1100), (2100, 2150)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
def test_one_matrix(lib, shape):
    for norm in NORMS:
        run(lib, [shape], [norm])


def test_matrices_of_all_sizes_at_once(lib):
    """each is held as its own size asks for"""
    run(lib, SHAPES, [NORMS[i % len(NORMS)] for i in range(len(SHAPES))])
    run(lib, [(128, 128)] * 9, NORMS)
    run(lib, [(1000, 1500)] * 6, [1e-3, 1e-8, 1e-12, 1.0, 1e-16, 1e-30])     # (tiles of the third product that are cut along k)


@pytest.mark.parametrize("steps", [1, 2, 9, 20, 64])
def test_numbers_of_steps(lib, steps):
    """as many steps as it takes to be large again (1e-12 grows by 3.4445^20 to 5e-2 of its own), and beyond: the result is held as the step before left it.  The bound
    lets an error grow 3.4445-fold in EVERY step, so what it says of many steps is little: those are compared with float32 as well"""
    shapes = [(60, 90), (100, 300), (160, 130)]
    for norm in (1e-9, 1e-14, 1e-25):
        run(lib, shapes, [norm] * 3, steps=steps)
    entries, n = om.lay_out(shapes)
    flat = torch.zeros(n, device="cuda")
    for i, v in enumerate(om.views(flat, entries)):
        v.copy_(small(*v.shape, 1e-16, i))
    out = torch.zeros(n, device="cuda")
    lib.orthogonalize(lib.MatrixPlan(entries), flat, out, steps=steps)
    for g, o in zip(om.views(flat, entries), om.views(out, entries)):
        want, single = om.iterate(g.double(), steps, EPS), om.iterate(g, steps, EPS).double()
        # an error in the direction of a singular value still small against one grows as the value itself does: relative to it, 2^-20 a step
        assert (o.double() - want).norm().item() <= max(4 * (single - want).norm().item(), (steps + 1) * om.STEP * want.norm().item())


@pytest.mark.parametrize("shape", [(2, 128), (128, 128), (100, 400), (333, 999), (1100, 1100)], ids=lambda s: f"{s[0]}x{s[1]}")
def test_16_bits(lib, shape):
    for norm in (1e-9, 1e-13):
        run(lib, [shape], [norm], "bf16")


def test_the_optimizer_step(lib):
    shapes = [(2, 128), (128, 128), (100, 400), (333, 999)]
    entries, n = om.lay_out(shapes)
    for norm in NORMS:
        g = torch.zeros(n, device="cuda")
        for i, v in enumerate(om.views(g, entries)):
            v.copy_(small(*v.shape, norm, i))
        w, m = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
        lib.muon_step(lib.MatrixPlan(entries), w, g, m, lr=0.5, momentum=0.0, nesterov=False, eps=EPS)
        for e, gv, wv in zip(entries, om.views(g, entries), om.views(w, entries)):
            check(wv / (-0.5 * e[4]), gv, 5, f"step of {e[1:3]}, norm {norm:g}")
