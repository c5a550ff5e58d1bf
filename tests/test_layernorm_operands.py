"""Layer norm's operands in one another's memory, and vectors off their float boundary: refused in front of any launch."""
import pytest
import torch

from encodermap_amd import _lib

P = 1 << 20    # addresses that nothing reads: every call here is refused in front of its launch
X, Y, DY, DX, G, B, M, R, DG, DB, W = (P * i for i in range(1, 12))
N, D = 4, 8    # 128 bytes of rows, 32 of columns, 16 of statistics


def fwd(**at):
    a = dict(x=X, y=Y, gamma=G, beta=B, mean=M, rstd=R)
    a.update(at)
    return _lib.load().emx_layernorm_fwd(a["x"], 0, N, D, D, a["gamma"], a["beta"], 1e-3, a["y"], D, a["mean"], a["rstd"], None)


def bwd(n=N, **at):
    a = dict(dy=DY, x=X, gamma=G, mean=M, rstd=R, dx=DX, dgamma=DG, dbeta=DB, ws=W)
    a.update(at)
    need = _lib.layernorm_ws_floats(n, D)
    return _lib.load().emx_layernorm_bwd(a["dy"], D, a["x"], D, 0, n, D, a["gamma"], a["mean"], a["rstd"], a["dx"], D, a["dgamma"], a["dbeta"], a["ws"], need, None)


@pytest.mark.parametrize("at", [
    dict(mean=R + 4), dict(rstd=M + 12), dict(mean=X), dict(mean=X + 124), dict(rstd=Y - 12), dict(mean=G + 28), dict(rstd=B), dict(y=G), dict(y=B - 124), dict(gamma=Y + 96),
    dict(gamma=G + 2), dict(beta=B + 1), dict(mean=M + 2), dict(rstd=R + 3),
])
def test_forward(at):
    assert fwd(**at) == -1
    assert b"emx_layernorm_fwd" in _lib.load().emx_last_error()


@pytest.mark.parametrize("at", [
    dict(dgamma=DB + 4), dict(dbeta=DG + 28), dict(dx=G), dict(dx=M - 124), dict(rstd=DX + 64), dict(ws=DY), dict(ws=X + 124), dict(ws=DX - 4), dict(ws=G), dict(ws=M), dict(ws=R + 8),
    dict(dgamma=W), dict(dbeta=W + 4), dict(dgamma=DX), dict(dbeta=DX + 100),
    dict(gamma=G + 2), dict(mean=M + 1), dict(rstd=R + 2), dict(dgamma=DG + 2), dict(dbeta=DB + 3), dict(ws=W + 2),
])
def test_backward(at):
    assert bwd(**at) == -1
    assert b"emx_layernorm_bwd" in _lib.load().emx_last_error()


def test_without_rows():
    assert bwd(n=0, dgamma=DB + 4) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("D", [70, 40000])
def test_sums_where_their_inputs_were(D):
    """dgamma and dbeta in the memory of gamma, mean, dy or x: written when those have been read"""
    _lib.require_gpu()
    n = 300
    gen = torch.Generator("cuda").manual_seed(D)
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x, dy, gamma = normal(n, D), normal(n, D), normal(D)
    y, mean, rstd = torch.empty_like(x), torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    _lib.layernorm_fwd(x, gamma, None, 1e-3, y, mean, rstd)
    ws = torch.empty(_lib.layernorm_ws_floats(n, D), device="cuda")
    want = [torch.empty_like(x), torch.empty(D, device="cuda"), torch.empty(D, device="cuda")]
    _lib.layernorm_bwd(dy, x, gamma, mean, rstd, *want, ws)
    for where in ("gamma", "rows"):
        xx, dd, gg, dx = x.clone(), dy.clone(), gamma.clone(), torch.empty_like(x)
        dg, db = (gg, dd[3]) if where == "gamma" else (xx[0], dd[n - 1])
        _lib.layernorm_bwd(dd, xx, gg, mean, rstd, dx, dg, db, ws)
        assert torch.equal(dx, want[0]) and torch.equal(dg, want[1]) and torch.equal(db, want[2]), where
