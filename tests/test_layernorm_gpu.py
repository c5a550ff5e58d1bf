"""Layer norm through the C ABI against its formula in 64 bits.

Tolerances.  u = 2^-24 is the unit roundoff of float32, e that of the rows' type (finfo(type).eps / 2).  A sum of D values by pairwise partial sums
of at most 64 terms carries a relative error of at most (64 + log2 D) u against the sum of magnitudes, here taken as 100 u (statistically a tenth of
it).  With the largest |x| / sigma of a row as k:
  mean    100 u max|x|                   (the mean's error is against the magnitudes that are added)
  rstd    200 u relative                 (a sum of squares, its square root and one reciprocal)
  y       e |y| + (200 + 100 k) u (|gamma| k + |beta|)   (the mean's error is seen through 1 / sigma)
  dx      e |dx| + (600 + 200 k) u rstd (max |t|) (1 + k^2)
  dgamma  sums over n rows: (100 + n) u is never reached -- 500 u sum |dy h| + the error of h: (200 + 100 k) u (1 + k) sum |dy|
  dbeta   500 u sum |dy|
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def lib():
    from encodermap_amd import _lib

    _lib.require_gpu()
    return _lib


def rows(n, D, dtype, pad, seed, offset=0.5):
    g = torch.Generator("cuda").manual_seed(seed)
    buf = torch.randn(n, D + pad, generator=g, device="cuda") * (0.25 + torch.rand(n, 1, generator=g, device="cuda")) + offset
    return buf.to(dtype)[:, :D], g


def blank(n, D, dtype, pad):
    """an output [n, D] inside a buffer of a value that must stay where it is"""
    buf = torch.full((n + 1, D + pad), 7.0, dtype=dtype, device="cuda")
    return buf, buf[:n, :D]


def untouched(buf, n, D):
    assert (buf[n:] == 7.0).all() and (buf[:, D:] == 7.0).all()


def formula(x, gamma, beta, eps):
    x = x.double()
    mu = x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x - mu).square().mean(1, keepdim=True) + eps)
    h = (x - mu) * rstd
    return mu, rstd, h, h * (1.0 if gamma is None else gamma.double()) + (0.0 if beta is None else beta.double())


def check(got, want, bound, what):
    err = (got.double() - want).abs()
    assert torch.isfinite(got.double()).all(), what
    worst = (err / bound.clamp_min(1e-300)).max().item() if err.numel() else 0.0
    assert (err <= bound).all(), f"{what}: {worst:.3g} of its bound, {err.max().item():.3g}"


def run_forward(lib, n, D, kind, pad, seed=0, gamma=True, beta=True, eps=1e-3, offset=0.5):
    dtype = TYPES[kind]
    e = torch.finfo(dtype).eps / 2
    x, g = rows(n, D, dtype, pad, seed, offset)
    gm = torch.randn(D, generator=g, device="cuda") if gamma else None
    bt = torch.randn(D, generator=g, device="cuda") if beta else None
    buf, y = blank(n, D, dtype, pad)
    mean, rstd = torch.full((n,), 3.0, device="cuda"), torch.full((n,), 3.0, device="cuda")
    lib.layernorm_fwd(x, gm, bt, eps, y, mean, rstd)
    mu64, rs64, h64, y64 = formula(x, gm, bt, eps)
    big = x.double().abs().amax(1, keepdim=True)
    k = (big * rs64).clamp_min(1.0)
    check(mean, mu64[:, 0], 100 * U * big[:, 0] + 1e-300, "mean")
    check(rstd, rs64[:, 0], (200 * U + 100 * U * k[:, 0]) * rs64[:, 0], "rstd")
    ga, ba = (1.0 if gm is None else gm.double().abs()), (0.0 if bt is None else bt.double().abs())
    check(y, y64, e * y64.abs() * (1 + 1e-3) + (200 + 100 * k) * U * (ga * k + ba) + torch.finfo(dtype).smallest_normal * e, "y")
    untouched(buf, n, D)
    return x, gm, mean, rstd, g, k


def run_backward(lib, n, D, kind, pad, seed=0, gamma=True, offset=0.5):
    dtype = TYPES[kind]
    e = torch.finfo(dtype).eps / 2
    x, gm, mean, rstd, g, k = run_forward(lib, n, D, kind, pad, seed, gamma=gamma, offset=offset)
    dy = torch.randn(n, D + pad, generator=g, device="cuda").to(dtype)[:, :D]
    buf, dx = blank(n, D, dtype, pad)
    dg, db = torch.full((D,), 5.0, device="cuda"), torch.full((D,), 5.0, device="cuda")
    ws = torch.full((lib.layernorm_ws_floats(n, D) + 1,), 9.0, device="cuda")
    lib.layernorm_bwd(dy, x, gm, mean, rstd, dx, dg, db, ws[:-1])
    _, rs64, h, _ = formula(x, gm, None, 1e-3)
    d64 = dy.double()
    t = d64 * (1.0 if gm is None else gm.double())
    want = rs64 * (t - t.mean(1, keepdim=True) - h * (t * h).mean(1, keepdim=True))
    top = t.abs().amax(1, keepdim=True)
    check(dx, want, e * want.abs() * (1 + 1e-3) + (600 + 200 * k) * U * rs64 * top * (1 + k * k) + torch.finfo(dtype).smallest_normal * e, "dx")
    check(dg, (d64 * h).sum(0), 500 * U * (d64 * h).abs().sum(0) + ((200 + 100 * k) * U * (1 + k) * d64.abs()).sum(0), "dgamma")
    check(db, d64.sum(0), 500 * U * d64.abs().sum(0), "dbeta")
    untouched(buf, n, D)
    assert ws[-1].item() == 9.0


WIDTHS = [1, 2, 3, 7, 8, 31, 32, 63, 64, 65, 127, 128, 129, 250, 256, 257, 500, 512, 515, 1000, 1024, 1025, 2047, 2048, 2850, 4096, 5000, 8191, 8192]


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("D", WIDTHS)
def test_widths(lib, D, kind):
    run_backward(lib, 37, D, kind, pad=0, seed=D)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("D", [16384, 16385, 32768, 40001, 65536, 70001, 150000])
def test_long_rows(lib, D, kind):
    run_backward(lib, 5, D, kind, pad=3, seed=D)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 15, 16, 17, 31, 63, 64, 65, 127, 255, 256, 257, 511, 513, 1000, 4096, 4097, 8191, 20000])
def test_row_counts(lib, n, kind):
    run_backward(lib, n, 128, kind, pad=0, seed=n)
    run_backward(lib, n, 70, kind, pad=1, seed=n)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("pad", [1, 2, 3, 5, 8, 16, 39])
def test_rows_inside_wider_ones(lib, pad, kind):
    run_backward(lib, 130, 200, kind, pad=pad, seed=pad)
    run_backward(lib, 33, 1537, kind, pad=pad, seed=pad)


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_rows_that_begin_anywhere(lib, kind):
    dtype = TYPES[kind]
    for at in range(1, 9):
        flat = torch.randn(20 * 67 + 16, generator=torch.Generator("cuda").manual_seed(at), device="cuda").to(dtype)
        x = flat[at:at + 20 * 67].view(20, 67)
        y = torch.zeros(20 * 67 + 16, dtype=dtype, device="cuda")[16 - at:16 - at + 20 * 67].view(20, 67)
        lib.layernorm_fwd(x, None, None, 1e-3, y)
        want = formula(x, None, None, 1e-3)[3]
        check(y, want, want.abs() * (1 + 1e-3) * (torch.finfo(dtype).eps / 2) + 2000 * U, f"offset {at}")


@pytest.mark.parametrize("gamma,beta", [(True, False), (False, True), (False, False)])
def test_without_weights(lib, gamma, beta):
    run_forward(lib, 50, 130, "f32", 0, gamma=gamma, beta=beta)
    run_backward(lib, 50, 130, "bf16", 0, gamma=gamma)


@pytest.mark.parametrize("offset", [0.0, 10.0, 300.0])
def test_rows_far_from_zero(lib, offset):
    run_backward(lib, 64, 384, "f32", 0, offset=offset)


def test_what_is_not_wanted_is_not_written(lib):
    n, D = 40, 96
    x, g = rows(n, D, torch.float32, 0, 3)
    dy = torch.randn(n, D, generator=g, device="cuda")
    gm = torch.randn(D, generator=g, device="cuda")
    y, mean, rstd = torch.empty(n, D, device="cuda"), torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    lib.layernorm_fwd(x, gm, None, 1e-3, y, mean, rstd)
    again = torch.empty_like(y)
    lib.layernorm_fwd(x, gm, None, 1e-3, again)
    assert torch.equal(y, again)
    ws = torch.empty(lib.layernorm_ws_floats(n, D), device="cuda")
    dx, dg, db = torch.empty(n, D, device="cuda"), torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
    lib.layernorm_bwd(dy, x, gm, mean, rstd, dx, dg, db, ws)
    dx2, dg2, db2 = torch.empty_like(dx), torch.empty_like(dg), torch.empty_like(db)
    lib.layernorm_bwd(dy, x, gm, mean, rstd, dx2, None, None)
    lib.layernorm_bwd(dy, x, gm, mean, rstd, None, dg2, None, ws)
    lib.layernorm_bwd(dy, x, gm, mean, rstd, None, None, db2, ws)
    tol = 1e-5   # (the passes that leave something out may add in another order)
    assert (dx - dx2).abs().max() <= tol * dx.abs().max() and (dg - dg2).abs().max() <= tol * dg.abs().max() and (db - db2).abs().max() <= tol * db.abs().max()


@pytest.mark.parametrize("D", [96, 2850, 20000])
def test_in_place(lib, D):
    n = 21
    x, g = rows(n, D, torch.float32, 4, 5)
    gm = torch.randn(D, generator=g, device="cuda")
    dy = torch.randn(n, D + 4, generator=g, device="cuda")[:, :D]
    y, mean, rstd = torch.empty_strided((n, D), (D + 4, 1), device="cuda"), torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    lib.layernorm_fwd(x, gm, None, 1e-3, y, mean, rstd)
    out = []
    for where in ("own", "dy", "x"):
        xs = torch.empty_strided((n, D), (D + 4, 1), device="cuda").copy_(x)
        dys = torch.empty_strided((n, D), (D + 4, 1), device="cuda").copy_(dy)
        dx = {"own": torch.empty_strided((n, D), (D + 4, 1), device="cuda"), "dy": dys, "x": xs}[where]
        dg, db = torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
        lib.layernorm_bwd(dys, xs, gm, mean, rstd, dx, dg, db, torch.empty(lib.layernorm_ws_floats(n, D), device="cuda"))
        out.append((dx.clone(), dg, db))
    for other in out[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out[0], other))
    z = torch.empty_strided((n, D), (D + 4, 1), device="cuda").copy_(x)
    lib.layernorm_fwd(z, gm, None, 1e-3, z)
    assert torch.equal(z, y)


def test_one_row_for_all(lib):
    """inputs broadcast over the rows (stride 0): the gradients are those of the rows written out"""
    n, D = 300, 200
    one, g = rows(1, D, torch.float32, 0, 9)
    x = one.expand(n, D)
    dy = torch.randn(1, D, generator=g, device="cuda").expand(n, D)
    res = []
    for xx, dd in ((x, dy), (x.contiguous(), dy.contiguous())):
        y, mean, rstd = torch.empty(n, D, device="cuda"), torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
        lib.layernorm_fwd(xx, None, None, 1e-3, y, mean, rstd)
        dx, dg, db = torch.empty(n, D, device="cuda"), torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
        lib.layernorm_bwd(dd, xx, None, mean, rstd, dx, dg, db, torch.empty(lib.layernorm_ws_floats(n, D), device="cuda"))
        res.append((y, dx, dg, db))
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_no_rows(lib):
    x = torch.empty(0, 12, device="cuda")
    none = torch.empty(0, device="cuda")
    lib.layernorm_fwd(x, None, None, 1e-3, torch.empty(0, 12, device="cuda"), none, none)
    dg, db = torch.ones(12, device="cuda"), torch.ones(12, device="cuda")
    lib.layernorm_bwd(x, x, None, none, none, torch.empty(0, 12, device="cuda"), dg, db, torch.empty(0, device="cuda"))
    assert (dg == 0).all() and (db == 0).all()


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("D", [70, 1500])
def test_a_row_that_is_not_finite_spoils_itself_alone(lib, D, value):
    x, _ = rows(30, D, torch.float32, 0, 2)
    clean = torch.empty_like(x)
    lib.layernorm_fwd(x, None, None, 1e-3, clean)
    x = x.clone()
    x[11, D // 2] = value
    y = torch.empty_like(x)
    lib.layernorm_fwd(x, None, None, 1e-3, y)
    keep = torch.arange(30, device="cuda") != 11
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[11]).any()


def test_constant_rows(lib):
    x = torch.full((5, 77), 3.25, device="cuda")
    y, mean, rstd = torch.empty_like(x), torch.empty(5, device="cuda"), torch.empty(5, device="cuda")
    beta = torch.randn(77, device="cuda")
    lib.layernorm_fwd(x, None, beta, 1e-3, y, mean, rstd)
    assert torch.allclose(y, beta.expand(5, 77), atol=77 * 3.25 * U * 32) and torch.allclose(rstd, torch.full_like(rstd, 1e-3 ** -0.5), rtol=1e-5)


def test_the_gradient_is_the_difference_quotient(lib):
    """sum(y w) moved along a direction: the change, in 64 bits, is the gradient's product with the direction"""
    n, D, eps = 9, 45, 1e-3
    x, g = rows(n, D, torch.float32, 0, 8)
    gm, bt = torch.randn(D, generator=g, device="cuda"), torch.randn(D, generator=g, device="cuda")
    w, v = torch.randn(n, D, generator=g, device="cuda"), torch.randn(n, D, generator=g, device="cuda")
    vg, vb = torch.randn(D, generator=g, device="cuda"), torch.randn(D, generator=g, device="cuda")
    y, mean, rstd = torch.empty(n, D, device="cuda"), torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    lib.layernorm_fwd(x, gm, bt, eps, y, mean, rstd)
    dx, dg, db = torch.empty(n, D, device="cuda"), torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
    lib.layernorm_bwd(w, x, gm, mean, rstd, dx, dg, db, torch.empty(lib.layernorm_ws_floats(n, D), device="cuda"))
    value = lambda s: (formula(x.double() + s * v.double(), gm.double() + s * vg.double(), bt.double() + s * vb.double(), eps)[3] * w.double()).sum()  # noqa: E731
    step = 1e-5   # a central difference: off by step^2 times the third derivative, ~1e-8 of the value here
    slope = ((value(step) - value(-step)) / (2 * step)).item()
    got = ((dx * v).double().sum() + (dg * vg).double().sum() + (db * vb).double().sum()).item()
    assert abs(got - slope) <= 1e-4 * ((dx * v).abs().sum() + (dg * vg).abs().sum() + (db * vb).abs().sum()).item()


def test_same_answer_every_time(lib):
    n, D = 3000, 333
    x, g = rows(n, D, torch.bfloat16, 0, 4)
    dy = torch.randn(n, D, generator=g, device="cuda").bfloat16()
    first = None
    for _ in range(3):
        y, mean, rstd = torch.empty_like(x), torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
        lib.layernorm_fwd(x, None, None, 1e-3, y, mean, rstd)
        dx, dg, db = torch.empty_like(x), torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
        lib.layernorm_bwd(dy, x, None, mean, rstd, dx, dg, db, torch.full((lib.layernorm_ws_floats(n, D),), float("nan"), device="cuda"))
        got = (y, mean, rstd, dx, dg, db)
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_on_another_stream_and_in_a_graph(lib):
    n, D = 700, 260
    x, g = rows(n, D, torch.float32, 0, 6)
    dy = torch.randn(n, D, generator=g, device="cuda")
    bufs = [torch.empty_like(x), torch.empty(n, device="cuda"), torch.empty(n, device="cuda"), torch.empty_like(x), torch.empty(D, device="cuda"),
            torch.empty(D, device="cuda")]
    ws = torch.empty(lib.layernorm_ws_floats(n, D), device="cuda")

    def step():
        y, mean, rstd, dx, dg, db = bufs
        lib.layernorm_fwd(x, None, None, 1e-3, y, mean, rstd)
        lib.layernorm_bwd(dy, x, None, mean, rstd, dx, dg, db, ws)

    step()
    want = [b.clone() for b in bufs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for b in bufs:
            b.zero_()
        step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(bufs, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(3):
        x.mul_(1.5)
        for b in bufs:
            b.zero_()
        graph.replay()
        torch.cuda.synchronize()
        replayed = [b.clone() for b in bufs]
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(bufs, replayed)), k


def test_refusals_of_the_binding(lib):
    x = torch.zeros(4, 8, device="cuda")
    y = torch.zeros(4, 8, device="cuda")
    bad = [
        lambda: lib.layernorm_fwd(x, None, None, 1e-3, torch.zeros(4, 9, device="cuda")),
        lambda: lib.layernorm_fwd(x, None, None, 1e-3, y.half()),
        lambda: lib.layernorm_fwd(x, None, None, 1e-3, torch.zeros(4, 8)),
        lambda: lib.layernorm_fwd(x[0], None, None, 1e-3, y[0]),
        lambda: lib.layernorm_fwd(x, torch.ones(7, device="cuda"), None, 1e-3, y),
        lambda: lib.layernorm_fwd(x, torch.ones(8, device="cuda").half(), None, 1e-3, y),
        lambda: lib.layernorm_fwd(x, torch.ones(16, device="cuda")[::2], None, 1e-3, y),
        lambda: lib.layernorm_fwd(x, None, None, 1e-3, y, mean=torch.zeros(3, device="cuda")),
        lambda: lib.layernorm_fwd(torch.zeros(8, 4, device="cuda").t(), None, None, 1e-3, y),
        lambda: lib.layernorm_fwd(x, None, None, 1e-3, torch.zeros(1, 8, device="cuda").expand(4, 8)),
        lambda: lib.layernorm_bwd(torch.zeros((), device="cuda").expand(4, 8), x, None, y[:, 0].contiguous(), y[:, 0].contiguous(), y, None, None),
        lambda: lib.layernorm_bwd(x, x, None, None, None, y, None, None),
        lambda: lib.layernorm_bwd(x, x, None, torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda"), y, torch.zeros(8, device="cuda"), None, None),
        lambda: lib.layernorm_bwd(x, x, None, torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda"), y, torch.zeros(8, device="cuda"), None,
                                  torch.zeros(1, device="cuda")),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(lib.EmxError):
            call()
            raise AssertionError(f"call {k} was accepted")
    assert (y == 0).all()
