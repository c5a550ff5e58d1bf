"""Layer norm step by step: every result against the formula in 64 bits on what the step HAS -- the statistics that the device has formed, not those of the exact
input -- so that a row's distance from zero is in the bound of its mean alone, and a term left out of a gradient is thousands of bounds away.  Each test says so itself:
it puts results with a planted mistake (made here, on the formula's side) to the same bound, which has to refuse them.

Tolerances, u = 2^-24 (one rounding to float32), e = finfo(type).eps / 2, worst case, nothing statistical.  A sum of a row is at most 32 values one after the other in
a thread (16 in the backward pass), six levels of a wave and sixteen waves: 54 roundings on the way of a term, 38 backward; longer rows go on in 64 bits.
  mean     54 u mean|x|, and the division's factor and product 2 u |mean|
  rstd     a square of a difference 3 u, its sum 54 u, the mean and eps 3 u: half of that through the root, then a root and a quotient, 3 u
  y        h = (x - mean) rstd two roundings, gamma and beta one more: 3 u |h gamma| + u |y|; e |y| stored
  dx       h: 2 u, t = dy gamma: u.  s = mean t: (38 + 1 + 2) u mean|t|;  q = mean t h: (38 + 4 + 2) u mean|t h|;
           rstd (t - (h q + s)): rstd (u |t| + |h| dq + 2 u |h q| + ds + u |h q + s| + 2 u |t - (h q + s)|), e |dx| stored
  dgamma   a column of a part is added one row after the other, then its groups and parts: (rows of a part + 32 + 5) u sum|dy h| + 2 u sum|dy h|
  dbeta    the same without the roundings of h
all times 1.01 for the products of errors."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-3
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def lib():
    from encodermap_amd import _lib

    _lib.require_gpu()
    return _lib


def held(got, want, bound, what):
    err = (got.double() - want).abs()
    assert torch.isfinite(got.double()).all(), what
    assert (err <= bound).all(), f"{what}: {(err / bound.clamp_min(1e-300)).max().item():.3g} of its bound"


def refused(planted, want, bound, what):
    """the bound sees the mistake, and not only in one place"""
    times = (planted.double() - want).abs() / bound.clamp_min(1e-300)
    assert times.median().item() > 10, f"{what}: {times.median().item():.3g} of the bound"


def run(lib, n, D, kind, offset, pad=0, seed=0):
    dtype = TYPES[kind]
    e, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    gen = torch.Generator("cuda").manual_seed(seed + D)
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x = (normal(n, D + pad) * (0.25 + torch.rand(n, 1, generator=gen, device="cuda")) + offset).to(dtype)[:, :D]
    gamma, beta = 1 + 0.3 * normal(D), 0.5 * normal(D)
    y, mean, rstd = torch.empty_like(x), torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    lib.layernorm_fwd(x, gamma, beta, EPS, y, mean, rstd)
    x64, g64, b64 = x.double(), gamma.double(), beta.double()
    mu = x64.mean(1)
    held(mean, mu, 1.01 * U * (54 * x64.abs().mean(1) + 2 * mu.abs()), "mean")
    m, r = mean.double()[:, None], rstd.double()[:, None]
    want = 1.0 / torch.sqrt((x64 - m).square().mean(1) + EPS)
    held(rstd, want, 1.01 * U * 33 * want, "rstd")
    h = (x64 - m) * r
    want = h * g64 + b64
    bound = 1.01 * (U * (3 * (h * g64).abs() + want.abs()) + e * want.abs()) + tiny
    held(y, want, bound, "y")
    if D > 2:
        refused(torch.zeros_like(want), want, bound, "y = 0")
        refused(want - b64, want, bound, "y without beta")
        refused(h + b64, want, bound, "y without gamma")
    # a gradient with a mean and a part along h: both sums of a row count
    dy = (normal(n, D + pad)[:, :D] + 0.5 + 0.5 * h.float()).to(dtype)
    dx, dgamma, dbeta = torch.empty_like(x), torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
    floats = lib.layernorm_ws_floats(n, D)
    lib.layernorm_bwd(dy, x, gamma, mean, rstd, dx, dgamma, dbeta, torch.empty(floats, device="cuda"))
    d64 = dy.double()
    t = d64 * g64
    s, q = t.mean(1, keepdim=True), (t * h).mean(1, keepdim=True)
    ds, dq = 41 * U * t.abs().mean(1, keepdim=True), 44 * U * (t * h).abs().mean(1, keepdim=True)
    join = h * q + s
    want = r * (t - join)
    bound = 1.01 * (r * (U * t.abs() + h.abs() * dq + 2 * U * (h * q).abs() + ds + U * join.abs() + 2 * U * (t - join).abs()) + e * want.abs()) + tiny
    held(dx, want, bound, "dx")
    if D > 2:
        refused(torch.zeros_like(want), want, bound, "dx = 0")
        if D > 64:      # (of few values, the part along h may be none)
            refused(r * (t - h * q), want, bound, "dx without the mean of t")
            refused(r * (t - s), want, bound, "dx without the part along h")
        refused(want / r, want, bound, "dx without rstd")
    parts = floats // (2 * D)
    depth = -(-n // parts) + 37
    size = (d64 * h).abs().sum(0)
    held(dgamma, (d64 * h).sum(0), 1.01 * U * (depth + 2) * size, "dgamma")
    held(dbeta, d64.sum(0), 1.01 * U * depth * d64.abs().sum(0), "dbeta")
    if D > 2 and n > 4:
        refused(torch.zeros_like(dgamma), (d64 * h).sum(0), 1.01 * U * (depth + 2) * size, "dgamma = 0")
        refused(torch.zeros_like(dbeta), d64.sum(0), 1.01 * U * depth * d64.abs().sum(0), "dbeta = 0")
        # (a row is 1 / n of `size`, half of them less than half of that; the bound is (depth + 2) u of it, 3.4e-6 at 57 roundings: ten times that up to n = 10^4)
        if n <= 10000:
            refused((d64 * h)[:-1].sum(0), (d64 * h).sum(0), 1.01 * U * (depth + 2) * size, "dgamma without the last row")


WIDTHS = [1, 2, 3, 33, 70, 128, 250, 512, 1000, 1024, 2048, 2850, 4096, 8191, 8192, 8193, 12288, 16383, 16384, 16385, 20000, 32768, 70001, 150000]


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("D", WIDTHS)
def test_widths(lib, D, kind):
    run(lib, 37, D, kind, 0.5, pad=D % 3)


@pytest.mark.parametrize("offset", [0.0, 10.0, 300.0, 1e4])
@pytest.mark.parametrize("D", [70, 384, 2850, 20000])
def test_rows_far_from_zero(lib, D, offset):
    run(lib, 64, D, "f32", offset)


@pytest.mark.parametrize("n", [1, 2, 9, 255, 4096, 20001])
def test_row_counts(lib, n):
    run(lib, n, 128, "f32", 0.5)
    run(lib, n, 300, "bf16", 0.5)


def test_few_long_rows(lib):
    run(lib, 2, 2 ** 21 + 3, "f32", 3.0)
    run(lib, 3, 2 ** 20 + 1, "bf16", 0.5)
