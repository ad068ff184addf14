"""The cases on which the Muon update, its orthogonalisation and the orthogonalisation's pullback are measured.

newton_schulz      y  = the odd quintic iteration X <- a X + (b X X^T + c (X X^T)^2) X on X / max(|X|_F, eps), five times, on the matrix's short side
newton_schulz_pullback   dx for a given dy, through every iteration and the normalisation
muon_raw           m <- beta m + (1 - beta) g;  u = beta m + (1 - beta) g (Nesterov);  p <- (1 - lr wd) p - lr s newton_schulz(u), for a list of weights at once

`own` chooses between elementary torch operations in 32 bits and the framework's own entry points."""
import math

import torch

own = False

COEF = (3.4445, -4.7750, 2.0315)
STEPS, EPS = 5, 1e-7
MUON = dict(lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.01, adjust="spectral", grad_scale=0.5)
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---- the cases ------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one 1x1 convolution of the ResNet-50 trunk's first stage: the smallest call, all latency
        dict(name="ns_64x64_f32", op="ns", batch=1, rows=64, cols=64, type="f32"),
        # a batch of odd matrices: no side is a multiple of a tile, a row of bf16 is not a multiple of 16 bytes
        dict(name="ns_5x97x211_bf16", op="ns", batch=5, rows=97, cols=211, type="bf16"),
        # the 512 -> 512 3x3 convolutions of the ResNet-18 trunk's last stage
        dict(name="ns_512x4608_f16", op="ns", batch=1, rows=512, cols=4608, type="f16"),
        # the expanding 1x1 convolutions of the ResNet-50 trunk's last stage: the short side is the columns
        dict(name="ns_2048x512_f32", op="ns", batch=1, rows=2048, cols=512, type="f32"),
        # a large dense weight: the largest call
        dict(name="ns_2048x8192_f32", op="ns", batch=1, rows=2048, cols=8192, type="f32"),
        # the pullback for an orthogonalised 3x3 convolution of the first stage, of the last stage's first, and for odd tall matrices
        dict(name="back_64x576_f32", op="back", batch=1, rows=64, cols=576, type="f32"),
        dict(name="back_512x2304_bf16", op="back", batch=1, rows=512, cols=2304, type="bf16"),
        dict(name="back_3x385x130_f16", op="back", batch=3, rows=385, cols=130, type="f16"),
        # the update of one weight
        dict(name="muon_128x1152", op="muon", shapes="128x1152"),
        # the updates of every hidden convolution of the depth and pose networks: one training step
        dict(name="muon_resnet18", op="muon", shapes="resnet18"),
        dict(name="muon_resnet50", op="muon", shapes="resnet50"),
        # odd weights packed one behind the other, so that most begin at an address that is a multiple of 4 bytes only; a row and a column among them
        dict(name="muon_odd", op="muon", shapes="37x53 1x700 129x65 300x1 255x257 64x63 17x1031 515x514"),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("ns", "back", "muon"))
    if op == "muon":
        if rng.random() < 0.5:                             # convolutions of a network of another width and depth
            shapes, c = [], rng.choice((16, 24, 32, 48, 80))
            for _ in range(rng.randint(2, 12)):
                o = rng.choice((c, 2 * c))
                shapes.append("%dx%d" % (o, c * rng.choice((1, 9))))
                c = min(o, 480)
        else:
            shapes = ["%dx%d" % (size(1, 900), size(1, 2500)) for _ in range(rng.randint(1, 20))]
        return dict(op=op, shapes=" ".join(shapes))
    most = 5.0e11 if op == "ns" else 1.0e11                # floating-point operations of the plain form
    while True:
        b, r, c = rng.choice((1, 1, 1, 2, 3, 8, 17)), size(1, 2600), size(1, 9000)
        if rng.random() < 0.4:
            r, c = -(-r // 32) * 32, -(-c // 32) * 32
        if op == "back" and r * c == 1:                   # its gradient is 0 and nothing else
            continue
        if STEPS * b * min(r, c) ** 2 * (4.0 * max(r, c) + 2.0 * min(r, c)) <= most:
            return dict(op=op, batch=b, rows=r, cols=c, type=rng.choice(("f32", "f32", "bf16", "f16")))


def _network(depth):
    """(rows, cols) of the hidden convolutions as matrices: the trunk without its stem, the depth decoder's branches, the pose decoder without its last layer."""
    got, cin = [], 64
    for planes, blocks in zip((64, 128, 256, 512), (2, 2, 2, 2) if depth == 18 else (3, 4, 6, 3)):
        out = planes if depth == 18 else 4 * planes
        for b in range(blocks):
            got += [(planes, 9 * cin), (planes, 9 * planes)] if depth == 18 else [(planes, cin), (planes, 9 * planes), (out, planes)]
            if b == 0 and (planes > 64 or cin != out):
                got.append((out, cin))
            cin = out
    top, skip = (512, (256, 128, 64, 64, 0)) if depth == 18 else (2048, (1024, 512, 256, 64, 0))
    inc = top
    for dec, s in zip((256, 128, 64, 32, 16), skip):
        got += [(dec, 9 * inc), (dec, 9 * (dec + s))]
        inc = dec
    return got + [(256, top), (256, 9 * 512), (256, 9 * 256)]


def _shapes(case):
    if case["op"] != "muon":
        return [(case["rows"], case["cols"])] * case["batch"]
    if case["shapes"].startswith("resnet"):
        return _network(int(case["shapes"][6:]))
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split()]


def work(case):
    """Each matrix product once, of a symmetric product one triangle; operands and results in the caller's types, once each."""
    size, flops, n = 0.0, 0.0, 0
    for r, c in _shapes(case):
        m, k = min(r, c), max(r, c)
        n += r * c
        forward = 3.0 * m * m * k + 1.0 * m * m * m         # X X^T (half of 2 m m k), A A (half of 2 m m m), B X
        # the pullback's step: G X^T (half suffices: only its symmetric part is used, but that takes both orders), S A, B G + V X, and X X^T, A A for B
        flops += STEPS * forward if case["op"] != "back" else STEPS * (forward + 2.0 * m * m * k + 2.0 * m * m * m + 4.0 * m * m * k) - 2.0 * m * m * k
    if case["op"] == "muon":
        size = 4.0 * 5 * n                                  # reads p, g, m; writes p, m
    else:
        size = (4 if case["type"] == "f32" else 2) * n * (2.0 if case["op"] == "ns" else 3.0)
    return {"bytes": size, "flops": flops}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _gradient(r, c, gen, scale=1e-3):
    """A gradient's spectrum: a few strong directions that decay, over a floor of noise."""
    k = min(r, c, 24)
    u = torch.randn(r, k, generator=gen, device="cuda") / torch.arange(1, k + 1, device="cuda").float()
    v = torch.randn(k, c, generator=gen, device="cuda")
    return scale * (u @ v + 0.3 * torch.randn(r, c, generator=gen, device="cuda"))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shapes = _shapes(case)
    if case["op"] != "muon":
        t = TYPES[case["type"]]
        state = {"op": case["op"], "x": torch.stack([_gradient(r, c, gen) for r, c in shapes]).to(t)}
        if case["op"] == "back":
            state["dout"] = torch.randn(state["x"].shape, generator=gen, device="cuda").to(t)
        return state
    n = sum(r * c for r, c in shapes)
    state = {"op": "muon", **{k: torch.empty(n, device="cuda") for k in ("p", "g", "m")}}
    at, views = 0, {k: [] for k in ("p", "g", "m")}
    for r, c in shapes:
        for k in views:
            views[k].append(state[k][at:at + r * c].view(r, c))
        views["p"][-1].uniform_(-1, 1, generator=gen).mul_(math.sqrt(6.0 / (r + c)))
        common = _gradient(r, c, gen, 2e-3)                 # what successive gradients share
        views["m"][-1].copy_(common + _gradient(r, c, gen, 5e-4))
        views["g"][-1].copy_(common + _gradient(r, c, gen, 2e-3))
        at += r * c
    return {**state, "params": views["p"], "grads": views["g"], "momenta": views["m"]}


# ---- one pass -------------------------------------------------------------------------------------------------------
def _iterates(x):
    """X / max(|X|_F, eps) with its short side first, and every iterate of it (32 bits; the norm, a long sum, in 64)."""
    a, b, c = COEF
    x = x.float()
    x = x / x.double().square().sum((-2, -1), keepdim=True).sqrt().clamp_min(EPS).float()
    x = x.mT.contiguous() if x.shape[-2] > x.shape[-1] else x
    xs = [x]
    for _ in range(STEPS):
        g = x @ x.mT
        x = a * x + (b * g + c * (g @ g)) @ x
        xs.append(x)
    return xs


def _back(x, dout):
    a, b, c = COEF
    tall = x.shape[-2] > x.shape[-1]
    xs, d = _iterates(x), dout.float()
    d = d.mT.contiguous() if tall else d
    for x_k in reversed(xs[:-1]):
        g = x_k @ x_k.mT
        s = d @ x_k.mT
        s = s + s.mT
        u = s @ g
        d = a * d + (b * g + c * (g @ g)) @ d + (b * s + c * (u + u.mT)) @ x_k
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt()
    along = (xs[0].double() * d.double()).sum((-2, -1), keepdim=True)
    d = torch.where(norm > EPS, d.double() - xs[0].double() * along, d.double()) / norm.clamp_min(EPS)
    return d.mT if tall else d


def run(state):
    if own:
        import md2amd
        md = md2amd.monodepth
        if state["op"] == "ns":
            return md.newton_schulz(state["x"], steps=STEPS, coefficients=COEF, eps=EPS)
        if state["op"] == "back":
            return md.newton_schulz_pullback(state["x"], state["dout"], steps=STEPS, coefficients=COEF, eps=EPS)
        md.muon_raw(state["params"], state["grads"], state["momenta"], steps=STEPS, coefficients=COEF, eps=EPS, **MUON)
        return state["p"], state["m"]
    if state["op"] == "ns":
        x = state["x"]
        y = _iterates(x)[-1]
        return (y.mT if x.shape[-2] > x.shape[-1] else y).to(x.dtype).contiguous()
    if state["op"] == "back":
        return _back(state["x"], state["dout"]).to(state["x"].dtype).contiguous()
    beta = MUON["momentum"]
    for p, g, m in zip(state["params"], state["grads"], state["momenta"]):
        g = MUON["grad_scale"] * g
        m.mul_(beta).add_(g, alpha=1 - beta)
        y = _iterates(beta * m + (1 - beta) * g)[-1]
        y = y.mT if p.shape[0] > p.shape[1] else y
        p.mul_(1 - MUON["lr"] * MUON["weight_decay"]).sub_(y, alpha=MUON["lr"] * math.sqrt(max(1.0, p.shape[0] / p.shape[1])))
    return state["p"], state["m"]


# ---- the same in 64 bits, from the definition -------------------------------------------------------------------------
def _exact_orthogonal(x):
    """The iteration acts on the singular values alone: U diag(f(f(..f(s / |s|)))) V^T is what it defines, computed here without a decomposition, on the side that X has."""
    x = x / torch.clamp(torch.linalg.matrix_norm(x), min=EPS)
    for _ in range(STEPS):
        if x.shape[0] <= x.shape[1]:
            q = x @ x.T
            x = COEF[0] * x + COEF[1] * (q @ x) + COEF[2] * (q @ (q @ x))
        else:
            q = x.T @ x
            x = COEF[0] * x + COEF[1] * (x @ q) + COEF[2] * ((x @ q) @ q)
    return x


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "ns":
        return torch.stack([_exact_orthogonal(x) for x in state["x"].double()])
    if case["op"] == "back":
        got = []
        for x, d in zip(state["x"].double(), state["dout"].double()):
            x.requires_grad_(True)
            got.append(torch.autograd.grad(_exact_orthogonal(x), x, d)[0])
        return torch.stack(got)
    ps, ms, beta = [], [], MUON["momentum"]
    for p, g, m in zip(state["params"], state["grads"], state["momenta"]):
        g = MUON["grad_scale"] * g.double()
        m = beta * m.double() + (1 - beta) * g
        y = _exact_orthogonal(beta * m + (1 - beta) * g)
        ms.append(m.flatten())
        ps.append(((1 - MUON["lr"] * MUON["weight_decay"]) * p.double() - MUON["lr"] * math.sqrt(max(1.0, p.shape[0] / p.shape[1])) * y).flatten())
    return torch.cat(ps), torch.cat(ms)
