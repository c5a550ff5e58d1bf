"""Layer norms between Dense layers, trained with the orthogonalised update: the pieces as a training loop uses them together -- the dense launches, layer
norm forward and backward, the weight gradients, emx_muon_step on the kernels, Adam on everything else, the operand stores rebuilt -- eagerly and
captured into one graph.

Each step is checked from the state the device has in front of it (float64, autograd): the loss to 1e-5; a gradient to 3e-4 of its largest entry (2e-5
for the dense launches, as their own tests hold them; a norm passes on (600 + 200 k) 2^-24 (1 + k^2) of the largest of its row, 1e-4 at k = 3, and
there are two on the way); momentum, kernels and the rest against the rule applied to the DEVICE's gradient, at the bounds of the operators' own tests.
"""
import math
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu

ABC = (3.4445, -4.7750, 2.0315)
B, EPS = 304, 1e-3
WIDTHS = [24, 96, 160, 24]
ACTS = [None, "tanh", None]
LR, MOMENTUM, DECAY, ADAM_LR, B1, B2, ADAM_EPS = 0.02, 0.95, 0.01, 1e-3, 0.9, 0.999, 1e-7


def orthogonal(g, steps=5, eps=1e-7):
    a, b, c = ABC
    x = g.t() if g.shape[0] > g.shape[1] else g
    x = x / (x.norm() + eps)
    for _ in range(steps):
        q = x @ x.t()
        x = a * x + (b * q + c * (q @ q)) @ x
    return x.t() if g.shape[0] > g.shape[1] else x


class Net:
    """x -> Dense -> norm -> Dense(tanh) -> norm -> Dense -> mean square against x; kernels in front of the flat buffer, the rest behind them"""

    def __init__(self, lib, seed=0):
        from encodermap_amd.layout import DenseSpec

        self.lib = lib
        gen = torch.Generator("cuda").manual_seed(seed)
        n = len(WIDTHS) - 1
        at, kernels = 0, []
        for i in range(n):
            kernels.append(at)
            at += WIDTHS[i] * WIDTHS[i + 1]
        self.tail = at
        biases, norms = [], []
        for i in range(n):
            biases.append(at)
            at += WIDTHS[i + 1]
        for i in range(n - 1):
            norms.append((at, at + WIDTHS[i + 1]))
            at += 2 * WIDTHS[i + 1]
        self.n = at
        self.specs = [DenseSpec(f"Dense_{i}", WIDTHS[i], WIDTHS[i + 1], ACTS[i], kernels[i], biases[i]) for i in range(n)]
        new = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
        self.w = new(at)
        for s in self.specs:
            self.w[s.w_off:s.w_off + s.n_in * s.n_out] = torch.randn(s.n_in * s.n_out, generator=gen, device="cuda") / math.sqrt(s.n_in)
            self.w[s.b_off:s.b_off + s.n_out] = 0.1 * torch.randn(s.n_out, generator=gen, device="cuda")
        for (g, b), width in zip(norms, WIDTHS[1:]):
            self.w[g:g + width] = 1 + 0.1 * torch.randn(width, generator=gen, device="cuda")
            self.w[b:b + width] = 0.1 * torch.randn(width, generator=gen, device="cuda")
        self.norms = norms
        self.g, self.m, self.v = new(at), new(at), new(at)
        self.x = torch.randn(B, WIDTHS[0], generator=gen, device="cuda")
        self.h = [new(B, k) for k in WIDTHS[1:]]          # outputs of the Dense layers
        self.y = [new(B, k) for k in WIDTHS[1:-1]]        # of the norms
        self.stats = [(new(B), new(B)) for _ in norms]
        self.delta = [new(B, k) for k in WIDTHS[1:]]
        self.dh = [new(B, k) for k in WIDTHS[1:]]         # d loss / d h
        self.dy = [new(B, k) for k in WIDTHS[1:-1]]
        self.loss = new(1)
        self.step_count = torch.zeros(1, dtype=torch.int64, device="cuda")
        self.red = new(lib.EMX_REDUCE_WS)
        # a Dense layer between two norms is a network of its own over the one parameter buffer
        self.plans = [lib.MlpPlan(SimpleNamespace(net_dim=s.n_in, layers=[s]), self.w, [self.h[i]], [self.delta[i]], train_rows=B)
                      for i, s in enumerate(self.specs)]
        self.wg = new(lib.mlp_wgrad_ws_floats(at, B))
        self.norm_ws = [new(lib.layernorm_ws_floats(B, k)) for k in WIDTHS[1:-1]]
        self.muon = lib.MatrixPlan.of_layers(self.specs)

    def part(self, flat, at, n):
        return flat[at:at + n]

    def step(self):
        lib, n = self.lib, len(self.specs)
        for i, plan in enumerate(self.plans):
            lib.mlp_forward(plan, 0, 1, self.x if i == 0 else self.y[i - 1], 0, B)
            if i < n - 1:
                (ga, be), k = self.norms[i], WIDTHS[i + 1]
                lib.layernorm_fwd(self.h[i], self.w[ga:ga + k], self.w[be:be + k], EPS, self.y[i], *self.stats[i])
        torch.sub(self.h[-1], self.x, out=self.dh[-1])
        self.loss.copy_(self.dh[-1].square().mean().reshape(1))
        self.dh[-1].mul_(2.0 / self.x.numel())
        for i in reversed(range(n)):
            lib.mlp_backward(self.plans[i], 0, 1, self.dh[i], None, 0, 0, B, dbelow=self.dy[i - 1] if i else None)
            lib.mlp_wgrad(self.plans[i], 0, 1, 0, B, self.g, self.wg)
            if i:
                (ga, be), k = self.norms[i - 1], WIDTHS[i]
                lib.layernorm_bwd(self.dy[i - 1], self.h[i - 1], self.w[ga:ga + k], *self.stats[i - 1], self.dh[i - 1], self.g[ga:ga + k],
                                  self.g[be:be + k], self.norm_ws[i - 1])
        lib.muon_step(self.muon, self.w, self.g, self.m, lr=LR, momentum=MOMENTUM, weight_decay=DECAY)
        rest = slice(self.tail, self.n)
        lib.adam_step(self.w[rest], self.g[rest], self.m[rest], self.v[rest], None, ADAM_LR, B1, B2, ADAM_EPS, None, self.step_count, None, self.red)
        self.step_count.add_(1)
        for plan in self.plans:
            plan.refresh_mirror()

    def state(self):
        return [t.clone() for t in (self.w, self.m, self.v, self.step_count)]

    def put(self, state):
        for t, s in zip((self.w, self.m, self.v, self.step_count), state):
            t.copy_(s)
        for plan in self.plans:
            plan.refresh_mirror()

    def autograd(self, w):
        """loss and gradient in float64 on the CPU from the flat weights ``w``"""
        w = w.double().cpu().requires_grad_(True)
        x = self.x.double().cpu()
        h = x
        for i, s in enumerate(self.specs):
            h = h @ w[s.w_off:s.w_off + s.n_in * s.n_out].view(s.n_in, s.n_out) + w[s.b_off:s.b_off + s.n_out]
            h = torch.tanh(h) if s.activation else h
            if i < len(self.specs) - 1:
                (ga, be), k = self.norms[i], s.n_out
                c = h - h.mean(1, keepdim=True)
                h = c / torch.sqrt(c.square().mean(1, keepdim=True) + EPS) * w[ga:ga + k] + w[be:be + k]
        loss = (h - x).square().mean()
        loss.backward()
        return loss.item(), w.grad


@pytest.fixture(scope="module")
def lib():
    from encodermap_amd import _lib

    _lib.require_gpu()
    return _lib


def test_steps_against_autograd(lib):
    net = Net(lib)
    u = 2.0 ** -24
    for t in range(1, 6):
        w0, m0, v0, _ = net.state()
        net.step()
        loss, grad = net.autograd(w0)
        assert abs(net.loss.item() - loss) <= 1e-5 * loss
        g = net.g.double().cpu()
        parts = [(s.w_off, s.n_in * s.n_out) for s in net.specs] + [(s.b_off, s.n_out) for s in net.specs] + \
                [(at, k) for pair, k in zip(net.norms, WIDTHS[1:]) for at in pair]
        for at, n in parts:
            top = grad[at:at + n].abs().max().item()
            assert (g[at:at + n] - grad[at:at + n]).abs().max().item() <= 3e-4 * top, (t, at, n)
        w0, m0, v0 = (a.double().cpu() for a in (w0, m0, v0))
        w, m, v = (a.double().cpu() for a in (net.w, net.m, net.v))
        for s in net.specs:
            part = slice(s.w_off, s.w_off + s.n_in * s.n_out)
            shape = (s.n_in, s.n_out)
            m64 = MOMENTUM * m0[part] + g[part]
            assert ((m[part] - m64).abs() <= 4 * u * (m0[part].abs() + g[part].abs())).all()
            direction = (g[part] + MOMENTUM * m64).view(shape)
            update, single = orthogonal(direction), orthogonal(direction.float()).double()
            scale = LR * max(1.0, s.n_out / s.n_in) ** 0.5
            want = (1 - LR * DECAY) * w0[part].view(shape) - scale * update
            err = (w[part].view(shape) - want).norm().item()
            side = min(shape)
            allowed = 2.0 ** -20 * sum(ABC[0] ** (5 - k) * min(ABC[0] ** k, 1.2024 * math.sqrt(side)) for k in range(6))
            allowed += 6 * u * 2 * (g[part].norm() + m64.norm()).item() / direction.norm().item() * ABC[0] ** 5
            assert err <= scale * allowed + 4 * u * want.norm().item()
            assert err <= scale * max(4 * (single - update).norm().item(), 8e-6 * update.norm().item()) + 4 * u * (want.norm() + w0[part].norm()).item()
        rest = slice(net.tail, net.n)
        m64 = m0[rest] + (g[rest] - m0[rest]) * (1 - B1)
        v64 = v0[rest] + (g[rest].square() - v0[rest]) * (1 - B2)
        want = w0[rest] - ADAM_LR * math.sqrt(1 - B2 ** t) / (1 - B1 ** t) * m64 / (v64.sqrt() + ADAM_EPS)
        assert (w[rest] - want).abs().max().item() <= 1e-5 * ADAM_LR * 10 + 2 * u * w0[rest].abs().max().item()


def test_the_whole_step_in_a_graph(lib):
    """replays, with eager steps of the same network between them, give the eager trajectory bit for bit"""
    net = Net(lib, seed=1)
    net.step()                                    # (what the library notes at first sight may not happen inside a capture)
    start = net.state()
    want = []
    for _ in range(4):
        net.step()
        torch.cuda.synchronize()
        want.append(net.state() + [net.loss.clone(), net.g.clone()])
    net.put(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        net.step()
    for k in range(4):
        if k == 2:                                # an eager step stands in for a replay
            net.step()
        else:
            graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(net.state() + [net.loss, net.g], want[k]):
            assert torch.equal(a, b), k
