"""Orthogonalised updates as a program calls them: over and over on one scratch whatever it holds, replayed on gradients of other sizes, two plans at once, more
matrices than one launch takes.  Every comparison is for equal bits."""
import pytest
import torch

from tests import test_muon_gpu as om

pytestmark = pytest.mark.gpu

# thin, small, low (one strip and several), 64 x 64 tiles, sums in parts, tiles cut along k
SHAPES = [(3, 90), (40, 50), (20, 300), (128, 128), (100, 700), (150, 130), (9000, 200), (1100, 1100)] + [(1000, 1500)] * 6


@pytest.fixture(scope="module")
def lib():
    from encodermap_amd import _lib

    _lib.require_gpu()
    return _lib


def gradients(shapes, seed, scale=1.0):
    entries, n = om.lay_out(shapes)
    flat = torch.zeros(n, device="cuda")
    for i, v in enumerate(om.views(flat, entries)):
        v.copy_(om.gradient(*v.shape, seed + i) * scale)
    return entries, flat


@pytest.mark.parametrize("scale", [1.0, 1e-12])
def test_any_content_of_the_scratch(lib, scale):
    for shapes in (SHAPES, SHAPES[:5], SHAPES[1:3], SHAPES[8:]):
        entries, g = gradients(shapes, 1, scale)
        plan = lib.MatrixPlan(entries)
        first = None
        for fill in (0, 255, 127, 60):
            plan.ws.fill_(fill)
            out = torch.zeros_like(g)
            lib.orthogonalize(plan, g, out)
            first = out if first is None else first
            assert torch.isfinite(out).all() and torch.equal(first, out), (len(shapes), fill)


def test_a_graph_replayed_on_gradients_of_other_sizes(lib):
    """what the step leaves in its scratch for its own later launches -- the norm, how X is held -- is the replay's, not the capture's"""
    entries, g0 = gradients(SHAPES[:8], 2)
    plan = lib.MatrixPlan(entries)
    g, w, m = g0.clone(), torch.zeros_like(g0), torch.zeros_like(g0)

    def step():
        lib.muon_step(plan, w, g, m, lr=0.1, momentum=0.5)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    scales = [1e-13, 1.0, 1e-9, 1e-20, 3.0]
    runs = []
    for how in (step, graph.replay):
        w.zero_(), m.zero_()
        got = []
        for s in scales:
            m.mul_(s)
            g.copy_(g0 * s)
            how()
            torch.cuda.synchronize()
            got.append((w.clone(), m.clone()))
        runs.append(got)
    for k, (a, b) in enumerate(zip(*runs)):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]), scales[k]


def test_two_plans_on_two_streams(lib):
    entries, g = gradients(SHAPES[:8], 3)
    plans = [lib.MatrixPlan(entries) for _ in range(2)]
    want = torch.zeros_like(g)
    lib.orthogonalize(plans[0], g, want)
    outs = [[torch.zeros_like(g) for _ in range(6)] for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for k in range(6):
        for p, s, o in zip(plans, streams, outs):
            with torch.cuda.stream(s):
                lib.orthogonalize(p, g, o[k])
    for s in streams:
        s.synchronize()
    assert all(torch.equal(o, want) for side in outs for o in side)


def test_an_optimizer_step_of_more_matrices_than_a_launch_takes(lib):
    """as many steps of one matrix each give the same"""
    shapes = [(5 + i % 60, 3 + i % 47) for i in range(110)]
    entries, g = gradients(shapes, 4)
    gen = torch.Generator("cuda").manual_seed(5)
    w0, m0 = torch.randn(g.numel(), generator=gen, device="cuda"), torch.randn(g.numel(), generator=gen, device="cuda") * 0.1
    w, m = w0.clone(), m0.clone()
    lib.muon_step(lib.MatrixPlan(entries), w, g, m, lr=0.05, weight_decay=0.1)
    w1, m1 = w0.clone(), m0.clone()
    for e in entries:
        lib.muon_step(lib.MatrixPlan([e]), w1, g, m1, lr=0.05, weight_decay=0.1)
    assert torch.equal(w, w1) and torch.equal(m, m1)
