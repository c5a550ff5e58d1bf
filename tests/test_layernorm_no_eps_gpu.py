"""Layer norm without an eps: ordinary rows need none.  A constant row has no spread to divide by: its own results mean nothing, and it spoils no other's."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("value", [0.0, 1.0, 1.1, 2.7])
@pytest.mark.parametrize("D", [3, 5, 7, 10, 130, 2850, 20000])
def test_a_constant_row_among_others(D, value):
    from encodermap_amd import _lib as lib

    lib.require_gpu()
    n = 12
    x = torch.randn(n, D, generator=torch.Generator("cuda").manual_seed(D), device="cuda")
    clean, y = torch.empty_like(x), torch.empty_like(x)
    mean, rstd = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    lib.layernorm_fwd(x, None, None, 0.0, clean, mean, rstd)
    m, r = mean.double()[:, None], rstd.double()[:, None]
    spread = (x.double() - m).square().mean(1).sqrt()
    assert ((rstd.double() * spread - 1).abs() <= 34 * U).all()           # (32 values a thread, six levels, sixteen waves: 60 u of a square, half of it, root and quotient)
    want = (x.double() - m) * r
    assert ((clean.double() - want).abs() <= 4 * U * want.abs()).all()
    x[5] = value
    lib.layernorm_fwd(x, None, None, 0.0, y, mean, rstd)
    keep = torch.arange(n, device="cuda") != 5
    assert torch.equal(y[keep], clean[keep])
    # D equal differences c over sqrt(c^2): the root of a mean of 60 roundings, where it is a number at all
    row = y[5][torch.isfinite(y[5])].double().abs()
    assert ((row - 1).abs() <= 64 * U).all()
    assert abs(mean[5].item() - value) <= 57 * U * value
