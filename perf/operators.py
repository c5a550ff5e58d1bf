"""The layer norm (forward, backward) and the orthogonalised matrix update (alone, and as a whole optimizer step): the cases they are measured on,
their plain forms in elementary torch operations, and the definition in 64 bits.

What a user of the framework trains is a stack of Dense layers whose kernels and biases lie in ONE flat float32 buffer, each kernel [n_in, n_out]
row-major and followed by its bias; the update's cases lay their matrices out the same way."""
import math
import random

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)   # of the quintic whose iteration drives singular values towards one
STEPS = 5
NORM_EPS = 1e-3        # the default of Keras' LayerNormalization
FROBENIUS_EPS = 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

# Dense kernels of the two networks that the benchmark trains: 128 features, and 512 angles (their sines and cosines: 1024 inputs)
NET_128 = "128x128,128x128,128x2,2x128,128x128,128x128"
NET_1024 = "1024x128,128x128,128x2,2x128,128x128,128x1024"


def listed():
    return [
        # a hidden layer's rows at the default batch: what one launch costs
        {"name": "norm_forward_256x128", "op": "norm_forward", "rows": 256, "width": 128, "type": "f32", "pad": 0},
        # odd rows, an odd width and rows that lie in a wider buffer, in 16 bits
        {"name": "norm_forward_10007x1001_bf16", "op": "norm_forward", "rows": 10007, "width": 1001, "type": "bf16", "pad": 39},
        # a whole resident training set (a million frames of 128 features) on its way through the encoder
        {"name": "norm_forward_1000000x128", "op": "norm_forward", "rows": 1000000, "width": 128, "type": "f32", "pad": 0},
        # the benchmark's training batch
        {"name": "norm_backward_4096x128", "op": "norm_backward", "rows": 4096, "width": 128, "type": "f32", "pad": 0},
        # the pair-distance features of a protein (2850 of them: rows that are not a multiple of 16 bytes)
        {"name": "norm_backward_2047x2850", "op": "norm_backward", "rows": 2047, "width": 2850, "type": "f32", "pad": 0},
        # a large batch of a wide layer, in 16 bits
        {"name": "norm_backward_65536x1024_bf16", "op": "norm_backward", "rows": 65536, "width": 1024, "type": "bf16", "pad": 0},
        # the kernels of one narrow network
        {"name": "orthogonalize_net_128", "op": "orthogonalize", "shapes": NET_128, "type": "f32", "pad": 0, "rank": 16},
        # half a dozen ragged matrices in 16 bits, rows inside wider ones
        {"name": "orthogonalize_6x1000x1500_bf16", "op": "orthogonalize", "shapes": ",".join(["1000x1500"] * 6), "type": "bf16", "pad": 4, "rank": 64},
        # one large square matrix
        {"name": "orthogonalize_4096x4096", "op": "orthogonalize", "shapes": "4096x4096", "type": "f32", "pad": 0, "rank": 64},
        # the optimizer step of the narrow network at batch 4096: the weight gradients arrive as 32 partial sums
        {"name": "muon_net_128", "op": "muon", "shapes": NET_128, "slices": 32, "nesterov": True, "rank": 16},
        # the same for the network with the wide ends
        {"name": "muon_net_1024", "op": "muon", "shapes": NET_1024, "slices": 32, "nesterov": True, "rank": 16},
        # a deep network of wide layers
        {"name": "muon_14_wide_layers", "op": "muon", "shapes": ",".join(["1024x4096"] + ["1024x1024"] * 12 + ["4096x1024"]), "slices": 1,
         "nesterov": False, "rank": 64},
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["norm_forward", "norm_backward", "orthogonalize", "muon"])
    if op.startswith("norm"):
        width = _log_uniform(rng, 8, 16384)
        kind = rng.choice(sorted(TYPES))
        rows = _log_uniform(rng, 1, min(1000000, max(1, 100000000 // width)))
        return {"op": op, "rows": rows, "width": width, "type": kind, "pad": rng.choice([0, 0, 8, rng.randrange(1, 40)])}
    while True:
        shapes = []
        for _ in range(rng.randrange(1, 5)):
            shape = "%dx%d" % (_log_uniform(rng, 1, 4096), _log_uniform(rng, 1, 4096))
            shapes += [shape] * rng.choice([1, 1, 2, 4])
        case = {"op": op, "shapes": ",".join(shapes), "rank": rng.choice([1, 8, 64, 256])}
        if op == "muon":
            case.update(slices=rng.choice([1, 1, 2, 7, 32]), nesterov=rng.random() < 0.5)
        else:
            case.update(type=rng.choice(sorted(TYPES)), pad=rng.choice([0, 0, 8, rng.randrange(1, 20)]))
        floats = sum(r * c for r, c in _shapes(case)) * case.get("slices", 1)
        if work(case)["flops"] <= 1.2e12 and floats <= 2 ** 27:
            return case


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _table(case):
    """(offset, rows, cols, row stride, update scale) of each kernel in the flat buffer, and the buffer's length; a bias follows every kernel and the
    next kernel begins at a multiple of 4"""
    out, at = [], 0
    for rows, cols in _shapes(case):
        ld = cols + case.get("pad", 0)
        out.append((at, rows, cols, ld, math.sqrt(max(1.0, cols / rows))))
        at += rows * ld + cols
        at = (at + 3) // 4 * 4
    return out, at


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(int(seed))
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    state = {"case": case}
    if own:
        from encodermap_amd import _lib

        state["lib"] = _lib
    if case["op"].startswith("norm"):
        rows, width, ld, kind = case["rows"], case["width"], case["width"] + case["pad"], TYPES[case["type"]]
        # activations of a Dense layer: a column mean of their own, rows of different spread
        x = (normal(rows, ld).mul_(normal(rows, 1).mul_(0.5).exp_()).add_(normal(1, ld).mul_(0.5))).to(kind)[:, :width]
        state.update(x=x, gamma=normal(width).mul_(0.1).add_(1.0), beta=normal(width).mul_(0.1))
        if case["op"] == "norm_forward":
            state["out"] = (torch.empty_strided((rows, width), (ld, 1), dtype=kind, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"))
        else:
            x64 = x.double()
            mean = x64.mean(1)
            state.update(mean=mean.float(), rstd=(x64 - mean[:, None]).square_().mean(1).add_(NORM_EPS).rsqrt_().float())
            state["dy"] = normal(rows, ld).mul_(0.1).to(kind)[:, :width]
            state["out"] = (torch.empty_strided((rows, width), (ld, 1), dtype=kind, device="cuda"), torch.empty(width, device="cuda"), torch.empty(width, device="cuda"))
            if own:
                state["ws"] = torch.empty(_lib.layernorm_ws_floats(rows, width), device="cuda")
        return state
    table, length = _table(case)

    def gradients(copies, scale):
        # sums over a batch of outer products: a few strong directions over a floor of weak ones, as weight gradients and their running means are
        flat = normal(copies, length).mul_(0.1 * scale)
        for at, rows, cols, ld, _ in table:
            r = min(case["rank"], rows, cols)
            strong = torch.linspace(0.0, -3.0, r, device="cuda").exp()
            u = normal(copies, rows, r).mul_(strong * scale / math.sqrt(r))
            flat[:, at:at + rows * ld].view(copies, rows, ld)[:, :, :cols] += torch.matmul(u, normal(1, r, cols).expand(copies, r, cols).contiguous())
        return flat

    state["table"] = table
    if case["op"] == "orthogonalize":
        kind = TYPES[case["type"]]
        state["g"] = gradients(1, 0.05)[0].to(kind)
        state["out"] = torch.zeros(length, dtype=kind, device="cuda")
    else:
        state["g"] = gradients(case["slices"], 0.05)
        state["m"] = gradients(1, 0.2)[0]
        state["w"] = normal(length).mul_(0.05)
    if own:
        state["plan"] = _lib.MatrixPlan(table, "cuda")
    return state


def run(state):
    case = state["case"]
    return {"norm_forward": _norm_forward, "norm_backward": _norm_backward, "orthogonalize": _orthogonalize, "muon": _muon}[case["op"]](case, state)


def _norm_forward(case, s):
    if own:
        y, mean, rstd = s["out"]
        s["lib"].layernorm_fwd(s["x"], s["gamma"], s["beta"], NORM_EPS, y, mean, rstd)
        return {"y": y, "mean": mean, "rstd": rstd}
    x = s["x"].float()
    mean = x.mean(1)
    centered = x - mean[:, None]
    rstd = torch.rsqrt(centered.square().mean(1) + NORM_EPS)
    y = centered * rstd[:, None] * s["gamma"] + s["beta"]
    return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}


def _norm_backward(case, s):
    if own:
        dx, dgamma, dbeta = s["out"]
        s["lib"].layernorm_bwd(s["dy"], s["x"], s["gamma"], s["mean"], s["rstd"], dx, dgamma, dbeta, s["ws"])
        return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xhat = (s["x"].float() - s["mean"][:, None]) * rstd
    t = dy * s["gamma"]
    dx = rstd * (t - t.mean(1, keepdim=True) - xhat * (t * xhat).mean(1, keepdim=True))
    return {"dx": dx.to(s["x"].dtype), "dgamma": (dy * xhat).sum(0), "dbeta": dy.sum(0)}


def _groups(table):
    """the matrices by shape: equal ones go through batched products together"""
    found = {}
    for entry in table:
        found.setdefault(entry[1:3], []).append(entry)
    return found


def _views(flat, entries):
    return [flat[at:at + rows * ld].view(rows, ld)[:, :cols] for at, rows, cols, ld, _ in entries]


def _iterate(x):
    """STEPS of the quintic iteration on a batch of matrices [k, rows, cols] in 32 bits"""
    a, b, c = COEFFICIENTS
    turned = x.shape[1] > x.shape[2]
    x = x.mT if turned else x
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + FROBENIUS_EPS)
    for _ in range(STEPS):
        gram = torch.matmul(x, x.mT)
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x.mT if turned else x


def _orthogonalize(case, s):
    if own:
        s["lib"].orthogonalize(s["plan"], s["g"], s["out"], steps=STEPS, eps=FROBENIUS_EPS)
        return {"out": _views(s["out"], s["table"])}
    made = {}
    for entries in _groups(s["table"]).values():
        for entry, o in zip(entries, _iterate(torch.stack(_views(s["g"], entries)).float())):
            made[entry[0]] = o.to(s["g"].dtype)
    return {"out": [made[entry[0]] for entry in s["table"]]}


def _muon(case, s):
    if own:
        s["lib"].muon_step(s["plan"], s["w"], s["g"], s["m"], lr=LR, momentum=MOMENTUM, nesterov=case["nesterov"], weight_decay=DECAY, steps=STEPS, eps=FROBENIUS_EPS)
        return {"w": s["w"], "m": s["m"]}
    total = s["g"].sum(0) if s["g"].shape[0] > 1 else s["g"][0]
    for entries in _groups(s["table"]).values():
        g = torch.stack(_views(total, entries))
        m = torch.stack(_views(s["m"], entries)).mul_(MOMENTUM).add_(g)
        o = _iterate(g + MOMENTUM * m if case["nesterov"] else m)
        for entry, w, kept, new, update in zip(entries, _views(s["w"], entries), _views(s["m"], entries), m, o):
            kept.copy_(new)
            w.mul_(1.0 - LR * DECAY).sub_(update, alpha=LR * entry[4])
    return {"w": s["w"], "m": s["m"]}


def work(case):
    if case["op"].startswith("norm"):
        n, d, size = case["rows"], case["width"], 4 if case["type"] == "f32" else 2
        forward = case["op"] == "norm_forward"
        return {"bytes": n * d * size * (2 if forward else 3) + 8 * n + (8 if forward else 12) * d, "flops": n * d * (8 if forward else 14)}
    flops = values = 0
    for rows, cols in _shapes(case):
        m, n = min(rows, cols), max(rows, cols)
        # one step: a symmetric product of m x n with itself, a symmetric one of m x m, a full m x m by m x n
        flops += STEPS * (m * m * n + m * m * m + 2 * m * m * n)
        values += rows * cols
    if case["op"] == "muon":
        return {"bytes": values * (16 + 4 * case["slices"]), "flops": flops}
    return {"bytes": values * 2 * (4 if case["type"] == "f32" else 2), "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("norm"):
        d = case["width"]
        x, gamma = s["x"].double(), s["gamma"].double()
        mu = x.sum(1, keepdim=True) / d
        sigma = ((x - mu).pow(2).sum(1, keepdim=True) / d + NORM_EPS).sqrt()
        z = (x - mu) / sigma
        if case["op"] == "norm_forward":
            return {"y": z * gamma + s["beta"].double(), "mean": mu[:, 0], "rstd": 1.0 / sigma[:, 0]}
        dy = s["dy"].double()
        dz = dy * gamma
        # d z_j / d x_i = (delta_ij - 1/d - z_i z_j / d) / sigma
        dx = (dz - (dz.sum(1, keepdim=True) + z * (dz * z).sum(1, keepdim=True)) / d) / sigma
        return {"dx": dx, "dgamma": (dy * z).sum(0), "dbeta": dy.sum(0)}
    a, b, c = COEFFICIENTS

    def polar(u):
        t = u if u.shape[0] <= u.shape[1] else u.t().contiguous()
        t = t / (torch.linalg.vector_norm(t) + FROBENIUS_EPS)
        for _ in range(STEPS):
            q = t @ t.t()
            p = q @ (c * q)
            p += b * q
            p.diagonal().add_(a)
            t = p @ t
        return t if u.shape[0] <= u.shape[1] else t.t()

    flat = s["g"].double()
    if case["op"] == "orthogonalize":
        return {"out": [polar(v) for v in _views(flat, s["table"])]}
    g, w, m = flat.sum(0), s["w"].double(), s["m"].double()
    for entry in s["table"]:
        (gv,), (wv,), (mv,) = (_views(t, [entry]) for t in (g, w, m))
        mv.copy_(MOMENTUM * mv + gv)
        wv.copy_((1.0 - LR * DECAY) * wv - LR * entry[4] * polar(gv + MOMENTUM * mv if case["nesterov"] else mv))
    return {"w": w, "m": m}
