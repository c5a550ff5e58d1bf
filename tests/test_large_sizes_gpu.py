"""Layer norm and orthogonalised updates at the upper end of what their entry points take: more threads than one launch has, rows of 2^27 values, columns
of 2^27 rows, matrices of the largest side.  Tolerances: those of test_layernorm_gpu.py and test_muon_gpu.py, whose derivations hold for any size."""
import math

import pytest
import torch

from tests import test_layernorm_gpu as ln
from tests import test_muon_gpu as om

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from encodermap_amd import _lib

    _lib.require_gpu()
    return _lib


@pytest.fixture(autouse=True)
def room(request):
    """these take tens of GB: nothing is left behind, and a smaller card skips them"""
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("less than 100 GB free")
    yield
    torch.cuda.empty_cache()


def test_rows_of_2_27_values(lib):
    ln.run_backward(lib, 2, 2 ** 27 + 5, "f16", pad=0, offset=3.0)


def test_more_rows_than_a_launch_has_threads_for(lib):
    """1024 threads to a row: 2^22 rows are 2^32 threads"""
    n, D, eps = 2 ** 22 + 3, 8200, 1e-3
    x = torch.empty(n, D, dtype=torch.bfloat16, device="cuda")
    some = torch.tensor([0, 1, 2 ** 21 - 1, 2 ** 21, 2 ** 21 + 1, 2 ** 22 - 1, 2 ** 22, n - 1], device="cuda")
    gen = torch.Generator("cuda").manual_seed(0)
    for r in range(0, n, 2 ** 17):
        x[r:r + 2 ** 17].normal_(0.5, 1.0, generator=gen)
    kept = x[some].clone()
    mean, rstd = torch.full((n,), 3.0, device="cuda"), torch.full((n,), 3.0, device="cuda")
    lib.layernorm_fwd(x, None, None, eps, x, mean, rstd)
    mu, rs, _, y = ln.formula(kept, None, None, eps)
    k = kept.double().abs().amax(1, keepdim=True) * rs
    e = torch.finfo(torch.bfloat16).eps / 2
    ln.check(mean[some], mu[:, 0], 100 * ln.U * kept.double().abs().amax(1), "mean")
    ln.check(rstd[some], rs[:, 0], (200 * ln.U + 100 * ln.U * k[:, 0]) * rs[:, 0], "rstd")
    ln.check(x[some], y, e * y.abs() * (1 + 1e-3) + (200 + 100 * k) * ln.U * k + torch.finfo(torch.bfloat16).smallest_normal * e, "y")
    # every row is normalised, once: 8200 values of deviation 1 around 0.5 are within 12 standard errors (0.011 and 0.0078) of that
    assert ((mean - 0.5).abs() < 0.14).all() and ((rstd - 1).abs() < 0.1).all()
    for r in range(0, n, 2 ** 17):
        assert (x[r:r + 2 ** 17].float().square().mean(1) - 1).abs().max().item() < 0.02     # (eps and the rounding to 8 bits: 0.001 + 2 x 2^-9)


def test_columns_of_2_27_rows(lib):
    """equal terms are the worst that a long sum can be given: their roundings all go one way"""
    n, D = 2 ** 27, 2
    gen = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(n, D, generator=gen, device="cuda")
    mean, rstd = torch.zeros(n, device="cuda"), torch.ones(n, device="cuda")
    dy = torch.full((1, D), 1.1, device="cuda")
    dg, db = torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
    ws = torch.empty(lib.layernorm_ws_floats(n, D), device="cuda")
    lib.layernorm_bwd(dy.expand(n, D), x, None, mean, rstd, None, dg, db, ws)
    one = dy[0].double()
    ln.check(db, n * one, 500 * ln.U * n * one, "dbeta")
    k = 6.0     # (the largest |x| of 2^28 normal ones)
    ln.check(dg, one * x.sum(0, dtype=torch.float64), 500 * ln.U * one * x.abs().sum(0, dtype=torch.float64) + (200 + 100 * k) * ln.U * (1 + k) * n * one, "dgamma")


def test_the_largest_matrix(lib):
    """G = (H x 1) diag(B_0 .. B_127): H the 128 x 128 matrix of signs whose rows are orthogonal, so that G has no zeros, orth(G) is
    (H / sqrt(128) x 1) diag(f(B_j)), and the formula is one of 256 x 256 matrices"""
    nb, s, steps, eps = 128, 256, 5, 1e-7
    side = nb * s
    sign = torch.ones(1, 1, device="cuda", dtype=torch.float64)
    for _ in range(7):
        sign = torch.cat([torch.cat([sign, sign], 1), torch.cat([sign, -sign], 1)], 0)
    gen = torch.Generator("cuda").manual_seed(2)
    b = torch.randn(nb, s, s, generator=gen, device="cuda")
    rows = b.permute(1, 0, 2)                                  # [r, j, c]
    g = torch.empty(nb, s, nb, s, device="cuda")
    for i in range(nb):
        g[i] = sign[i].float()[None, :, None] * rows
    out = torch.full((side * side + 8,), 7.0, device="cuda")
    plan = lib.MatrixPlan([(0, side, side, side, 1.0)])
    lib.orthogonalize(plan, g.view(-1), out, steps=steps, eps=eps)
    norm = math.sqrt(nb) * b.double().square().sum().sqrt() + eps
    f = torch.empty(nb, s, s, dtype=torch.float64, device="cuda")
    a1, a3, a5 = om.ABC
    for j in range(nb):
        x = b[j].double() * (math.sqrt(nb) / norm)
        for _ in range(steps):
            gram = x @ x.t().contiguous()
            x = a1 * x + (a3 * gram + a5 * (gram @ gram)) @ x
        f[j] = x
    rows64 = f.permute(1, 0, 2)
    off = torch.zeros((), dtype=torch.float64, device="cuda")
    res = out[:side * side].view(nb, s, nb, s)
    for i in range(nb):
        off += (res[i].double() - (sign[i] / math.sqrt(nb))[None, :, None] * rows64).square().sum()
    assert torch.isfinite(off) and (out[side * side:] == 7.0).all()
    limit = om.bound(side, side, steps)
    assert off.sqrt().item() <= limit, f"{off.sqrt().item():.3g} off, {limit:.3g} allowed of {f.norm().item():.3g}"


def test_what_an_int_does_not_hold_is_refused(lib):
    x = torch.empty(1, 2 ** 32 + 8, dtype=torch.float16, device="cuda")
    with pytest.raises(lib.EmxError, match="values"):
        lib.layernorm_fwd(x, None, None, 1e-3, x)
    g = torch.zeros(64, device="cuda")
    plan = lib.MatrixPlan([(0, 8, 8, 8, 1.0)])
    with pytest.raises(lib.EmxError, match="steps"):
        lib.orthogonalize(plan, g, g, steps=2 ** 32 + 5)
    with pytest.raises(lib.EmxError, match="steps"):
        lib.muon_step(plan, g.clone(), g, g.clone(), lr=0.1, steps=2 ** 32 + 5)
    parts = torch.zeros(2 ** 31, 1, device="cuda")
    with pytest.raises(lib.EmxError, match="slices"):
        lib.muon_step(lib.MatrixPlan([(0, 1, 1, 1, 1.0)]), g.clone(), parts, g.clone(), lr=0.1)
