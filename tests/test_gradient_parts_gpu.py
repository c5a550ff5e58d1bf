"""The optimizer step on a gradient that arrives as parts: what a sum of them is off by, and the parts as emx_mlp_wgrad leaves them.

With no momentum and a momentum buffer of zeros, that buffer is the sum itself.  Tolerances.  u = 2^-24.  A sum of parts of equal spread rounds each partial sum of k
parts once, by a variance of k: 2 + 3 + ... + n = 527 for 32 parts one after the other, n log2 n = 160 for a tree, 24 (three levels of eight) for each eight and 8 k for
the sum of k of those: 168 for 32 parts, at most 1.06 times the tree's root for 8 ... 32 parts (31: seven of them in a row), 1.23 times for 100.  1.3 times the error
of a tree is allowed; one after the other is 1.8 times at 32 parts, 1.4 at 16 and no more than 1.3 below 12."""
import pytest
import torch

from tests import test_muon_gpu as om

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def lib():
    from encodermap_amd import _lib

    _lib.require_gpu()
    return _lib


def tree(parts):
    while parts.shape[0] > 1:
        even = parts[0:parts.shape[0] // 2 * 2:2] + parts[1::2]
        parts = torch.cat([even, parts[-1:]]) if parts.shape[0] % 2 else even
    return parts[0]


@pytest.mark.parametrize("cols", [256, 255])          # (four elements to a thread at a time; one)
@pytest.mark.parametrize("parts", [1, 2, 7, 8, 9, 12, 16, 24, 31, 32, 100])
def test_the_sum_is_as_exact_as_a_tree(lib, parts, cols):
    rows = 300
    n = rows * cols
    g = torch.randn(parts, n, generator=torch.Generator("cuda").manual_seed(parts), device="cuda")
    w, m = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    lib.muon_step(lib.MatrixPlan([(0, rows, cols, cols, 1.0)]), w, g, m, lr=0.1, momentum=0.0)
    want = g.double().sum(0)
    err, plain = (m.double() - want).norm().item(), (tree(g).double() - want).norm().item()
    assert ((m.double() - want).abs() <= parts * U * g.double().abs().sum(0)).all()
    assert err <= 1.3 * plain, f"{err / want.norm().item():.3g} off, a tree {plain / want.norm().item():.3g}"


@pytest.mark.parametrize("rows", [4096, 3000, 77])
def test_the_parts_that_the_dense_layers_leave(lib, rows):
    """emx_mlp_wgrad without a gradient to write: its scratch IS the parts, of the kernels and of the biases between them"""
    from encodermap_amd.layout import build_layout, init_parameters

    lay = build_layout([96, 64, 2], ["", "tanh", "tanh", ""], 60)
    n = lay.n_params
    gen = torch.Generator("cuda").manual_seed(rows)
    params = torch.from_numpy(init_parameters(lay, 2)).cuda()
    x = torch.randn(rows, 60, generator=gen, device="cuda")
    h = [torch.zeros(rows, s.n_out, device="cuda") for s in lay.layers]
    delta = [torch.zeros(rows, s.n_out, device="cuda") for s in lay.layers]
    net = lib.MlpPlan(lay, params, h, delta, train_rows=rows)
    layers = len(lay.layers)
    lib.mlp_forward(net, 0, layers, x, 0, rows)
    lib.mlp_backward(net, 0, layers, (h[-1] - x) / rows, None, 0, 0, rows)
    ws = torch.zeros(lib.mlp_wgrad_ws_floats(n, rows), device="cuda")
    lib.mlp_wgrad(net, 0, layers, 0, rows, None, ws)
    slices = lib.mlp_wgrad_slices(rows)
    parts = ws[:slices * n].view(slices, n)
    whole, other = torch.zeros(n, device="cuda"), torch.zeros_like(ws)
    lib.mlp_wgrad(net, 0, layers, 0, rows, whole, other)
    plan = lib.MatrixPlan.of_layers(lay.layers)
    before = parts.clone()
    w, m = params.clone(), torch.zeros(n, device="cuda")
    lib.muon_step(plan, w, parts, m, lr=0.02, momentum=0.0)
    w1, m1 = params.clone(), torch.zeros(n, device="cuda")
    lib.muon_step(plan, w1, whole, m1, lr=0.02, momentum=0.0)
    assert torch.equal(parts, before)
    total, size = parts.double().sum(0), parts.double().abs().sum(0)
    kernels = torch.zeros(n, dtype=torch.bool, device="cuda")
    for s in lay.layers:
        part = slice(s.w_off, s.w_off + s.n_in * s.n_out)
        kernels[part] = True
        assert total[part].abs().max() > 0
        assert ((m[part].double() - total[part]).abs() <= slices * U * size[part]).all()
        # and it is the gradient: the same sum in emx_mlp_wgrad's own order
        assert ((m[part] - whole[part]).abs() <= 2 * slices * U * size[part]).all()
        shape = (s.n_in, s.n_out)
        update = om.iterate(total[part].view(shape))
        moved = (params[part] - w[part]).view(shape).double()
        scale = 0.02 * max(1.0, s.n_out / s.n_in) ** 0.5
        # an error of the sum, slices u of the magnitudes, is one of X_0 and grows 3.4445^5-fold at most
        start = slices * U * (size[part].norm() / total[part].norm()).item() * om.ABC[0] ** 5
        limit = scale * (om.bound(*shape, 5) + start) + 2 * U * (params[part].double().norm().item() + scale * update.norm().item())
        assert (moved - scale * update).norm().item() <= limit
    assert torch.equal(w[~kernels], params[~kernels]) and (m[~kernels] == 0).all()      # biases, and what lies between the tensors
