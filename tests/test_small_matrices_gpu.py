"""Orthogonalisation of small matrices: as exact as float32, whatever their singular values.

Those of 17 to 48 rows run on float32 operands, and round where the plain iteration in float32 does: the root mean square of their errors over a set of matrices is
that of the plain iteration's (1), but for the order of the sums.  1.2 times it is allowed over 24 matrices; operands of 22 bits, rounded twice, make up to 2^0.5 times
it, less as the sums get longer: from 49 rows on the sums' own roundings are the larger part."""
import math

import pytest
import torch

from tests import test_muon_gpu as om

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from encodermap_amd import _lib

    _lib.require_gpu()
    return _lib


def noise(rows, cols, seed):
    return torch.randn(rows, cols, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")


def errors(lib, shapes, make):
    """root mean square of the relative errors: here, and of the iteration in float32"""
    entries, n = om.lay_out(shapes)
    flat = torch.zeros(n, device="cuda")
    for i, v in enumerate(om.views(flat, entries)):
        v.copy_(make(*v.shape, i))
    out = torch.zeros(n, device="cuda")
    lib.orthogonalize(lib.MatrixPlan(entries), flat, out)
    own, plain = [], []
    for g, o in zip(om.views(flat, entries), om.views(out, entries)):
        want = om.iterate(g.double())
        own.append(((o.double() - want).norm() / want.norm()).item())
        plain.append(((om.iterate(g.contiguous()).double() - want).norm() / want.norm()).item())
    rms = lambda v: math.sqrt(sum(e * e for e in v) / len(v))  # noqa: E731
    return rms(own), rms(plain)


@pytest.mark.parametrize("make", [noise, om.gradient], ids=["noise", "gradient"])
@pytest.mark.parametrize("rows,cols", [(17, 17), (18, 60), (20, 96), (24, 300), (31, 128), (32, 33), (33, 70), (40, 128), (48, 48), (50, 900), (63, 65), (64, 128), (17, 5000)])
def test_as_exact_as_float32(lib, rows, cols, make):
    for shape in ((rows, cols), (cols, rows)):
        own, plain = errors(lib, [shape] * 24, make)
        assert own <= 1.2 * plain, f"{shape}: {own:.3g}, float32 {plain:.3g}"


@pytest.mark.parametrize("rows", list(range(15, 68)))
def test_every_number_of_rows(lib, rows):
    """(the padding of a block of 16 rows or columns, one strip and several)"""
    om.orthogonalize(lib, [(rows, rows + 1), (rows, 130), (300, rows), (rows, rows)], seed=rows)
    om.orthogonalize(lib, [(rows, 100), (127, rows)], "bf16", pad=3, seed=rows)
    om.muon_case(lib, [(rows, 90), (200, rows)], 3, True, 0.05, seed=rows, pad=1)
