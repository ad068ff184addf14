"""Muon: newton_schulz, newton_schulz_pullback and muon_raw against plain implementations in 64 bits, their refusals (host logic, no GPU), and the ways they are called.

Tolerances.  Inside, a matrix element is a pair of f16 (off by at most 2^-22 of its value) and a product drops lo * lo (2^-22 again): a step's operands put at most e = 3 * 2^-22 of the
iterate's norm into the next iterate, which later steps amplify by at most a = 3.4445 each.  Summed over five steps that is e * a^5 / (a - 1) = 1.4e-4 per singular direction, where a
result of full rank has singular values of 0.68 and more: 2.1e-4 of the result's norm in the worst case (LOOSE).  Roundings do not all point one way: the error is also held to twice
that of the same formulas in plain fp32, with a floor of 2e-6 (a few 2^-24 through a^5 = 485, averaged over the directions)."""
import ctypes
import math

import numpy as np
import pytest
import torch

import md2amd

gpu = pytest.mark.gpu
LOOSE = 2.1e-4
HALF = {torch.float32: 0.0, torch.bfloat16: torch.finfo(torch.bfloat16).eps / 2, torch.float16: torch.finfo(torch.float16).eps / 2}
COEF = (3.4445, -4.7750, 2.0315)


def md():
    return md2amd.monodepth


def ns_plain(x, steps=5, coef=COEF, eps=1e-7):
    """The definition, in x's type (the norm in 64 bits), for (..., rows, cols)."""
    a, b, c = coef
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt().clamp_min(eps)
    x = (x.double() / norm).to(x.dtype)
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2).contiguous() if tall else x
    for _ in range(steps):
        g = x @ x.transpose(-1, -2).contiguous()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.transpose(-1, -2) if tall else x


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / (b.norm() + 1e-300))


def gradient_like(shape, seed, noise=0.3, scale=1e-3):
    g = torch.Generator().manual_seed(seed); r, c = shape[-2:]; k = min(r, c, 8); lead = tuple(shape[:-2])
    u = torch.randn(lead + (r, k), generator=g, dtype=torch.float64) / torch.arange(1, k + 1)
    return scale * (u @ torch.randn(lead + (k, c), generator=g, dtype=torch.float64) + noise * torch.randn(tuple(shape), generator=g, dtype=torch.float64))


# ---- refusals: decided on the host, before anything reaches the GPU ---------------------------------------------------------
def last_error():
    return md2amd._lib.lib().md2_last_error(None).decode()


def test_tensors_that_are_refused():
    m = md()
    for bad in (torch.zeros(4, 4), torch.zeros(4), [[1.0]], torch.zeros(4, 4, dtype=torch.float64)):
        with pytest.raises(ValueError):
            m.newton_schulz(bad)
    with pytest.raises(ValueError):
        m.newton_schulz_pullback(torch.zeros(4, 4), torch.zeros(4, 4))
    with pytest.raises(ValueError):
        m.muon_raw([torch.zeros(4, 4)], [torch.zeros(4, 4)], [torch.zeros(4, 4)])
    with pytest.raises(ValueError):
        m.muon_raw([torch.zeros(4, 4)], [], [torch.zeros(4, 4)])
    with pytest.raises(ValueError):
        m.muon_raw([], [], [], adjust="other")


def test_workspace_sizes_and_refused_sizes():
    L = md2amd._lib.lib()
    for pull in (0, 1):
        assert L.md2_newton_schulz_workspace(1, 1, 1, 5, pull) > 0
        for bad in ((0, 4, 4), (1, 0, 4), (1, 4, 0), (-1, 4, 4), (1, -4, 4), (1, 1 << 21, 4), (1, 1 << 17, 1 << 17), (1 << 21, 4, 4)):
            assert L.md2_newton_schulz_workspace(*bad, 5, pull) == -1, bad
        for steps in (0, -1, 17):
            assert L.md2_newton_schulz_workspace(1, 4, 4, steps, pull) == -1
    assert L.md2_newton_schulz_workspace(3, 100, 200, 5, 0) < L.md2_newton_schulz_workspace(3, 100, 200, 5, 1)
    I = ctypes.c_int64
    assert L.md2_muon_workspace((I * 2)(3, 4), (I * 2)(5, 6), 2, 5) > 0 and L.md2_muon_workspace((I * 1)(3), (I * 1)(0), 1, 5) == -1 and L.md2_muon_workspace(None, None, 1, 5) == -1


def ns_c(x=4096, y=8192, batch=1, rows=8, cols=8, strides=(64, 8, 1), dtype=0, steps=5, coef=COEF, eps=1e-7, ws=4096, nbytes=None):
    L = md2amd._lib.lib()
    st = (ctypes.c_int64 * 3)(*strides) if strides else None; co = (ctypes.c_double * 3)(*coef) if coef else None
    return L.md2_newton_schulz(x, y, batch, rows, cols, st, dtype, steps, co, eps, ws, 0 if nbytes is None else nbytes, None)


@pytest.mark.parametrize("kw,word", [
    (dict(strides=None), "strides"), (dict(coef=None), "coefficients"), (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(steps=0), "steps"), (dict(steps=17), "steps"),
    (dict(eps=0.0), "eps"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(eps=math.inf), "eps"), (dict(coef=(math.nan, 0, 0)), "finite"), (dict(coef=(9.0, 0, 0)), "past 4"),
    (dict(coef=(3.4445, -4.775, 200.0)), "past"), (dict(x=None), "null"), (dict(y=None), "null"), (dict(rows=0), "sizes"), (dict(cols=-3), "sizes"), (dict(x=4097), "aligned"),
    (dict(strides=(64, -8, 1)), "stride"), (dict(ws=None), "workspace"), (dict(), "workspace"), (dict(ws=4100, nbytes=1 << 40), "workspace")])
def test_newton_schulz_refuses(kw, word):
    """Every one of these is found before the first launch (the pointers are never followed): status 2 and a reason."""
    assert ns_c(**kw) == 2 and word in last_error(), (kw, last_error())


def test_pullback_refuses_steps_that_would_leave_the_range():
    L = md2amd._lib.lib(); st = (ctypes.c_int64 * 3)(64, 8, 1); co = (ctypes.c_double * 3)(*COEF)
    assert L.md2_newton_schulz_bwd(4096, 4096, 8192, 1, 8, 8, st, st, 0, 12, co, 1e-7, 4096, 0, None) == 2 and "pullback" in last_error()
    assert L.md2_newton_schulz_bwd(4096, None, 8192, 1, 8, 8, st, st, 0, 5, co, 1e-7, 4096, 0, None) == 2 and "null" in last_error()
    assert L.md2_newton_schulz_bwd(4096, 4096, 8192, 1, 8, 8, st, None, 0, 5, co, 1e-7, 4096, 0, None) == 2 and "strides" in last_error()


def muon_c(p=(4096,), g=(8192,), m=(16384,), rows=(8,), cols=(8,), lr=0.02, momentum=0.95, decay=0.0, adjust=0, scale=1.0, steps=5, eps=1e-7, count=None):
    L = md2amd._lib.lib(); n = len(p); V, I = ctypes.c_void_p, ctypes.c_int64
    return L.md2_muon_raw((V * n)(*p), (V * n)(*g), (V * n)(*m), (I * n)(*rows), (I * n)(*cols), n if count is None else count, lr, momentum, 1, decay, adjust, scale, steps,
                          (ctypes.c_double * 3)(*COEF), eps, 4096, 0, None)


@pytest.mark.parametrize("kw,word", [
    (dict(count=0), "no weights"), (dict(rows=(0,)), "sizes"), (dict(lr=-1.0), "lr"), (dict(lr=math.nan), "lr"), (dict(momentum=1.0), "momentum"), (dict(momentum=-0.1), "momentum"),
    (dict(decay=-1.0), "weight_decay"), (dict(decay=math.inf), "weight_decay"), (dict(adjust=2), "adjust"), (dict(scale=math.nan), "grad_scale"), (dict(steps=0), "steps"), (dict(eps=0.0), "eps"),
    (dict(p=(None,)), "null"), (dict(p=(4098,)), "aligned"), (dict(), "workspace"),
    (dict(p=(4096,), m=(4096,)), "overlaps"), (dict(p=(4096,), g=(4096 + 252,)), "overlaps"), (dict(m=(8192,)), "overlaps"),
    (dict(p=(4096, 4096), g=(8192, 8192), m=(16384, 20480), rows=(8, 8), cols=(8, 8)), "overlaps"),
    (dict(p=(4096, 4096 + 128), g=(8192, 8192), m=(16384, 20480), rows=(8, 8), cols=(8, 8)), "overlaps")])
def test_muon_raw_refuses(kw, word):
    assert muon_c(**kw) == 2 and word in last_error(), (kw, last_error())


def test_two_weights_may_share_a_gradient():
    """Only what the step writes has to be disjoint: the next refusal is the workspace's."""
    assert muon_c(p=(4096, 4096 + 256), g=(8192, 8192), m=(16384, 20480), rows=(8, 8), cols=(8, 8)) == 2 and "workspace" in last_error()


# ---- newton_schulz ------------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1), (1, 7), (9, 1), (2, 2), (16, 16), (31, 33), (64, 64), (65, 64), (64, 576), (127, 130), (128, 128), (129, 129), (200, 77), (33, 1000), (130, 300), (257, 96), (256, 640), (385, 514),
          (32, 1152), (32, 1153), (1153, 20), (64, 512), (513, 64), (61, 575), (577, 64), (32, 1185), (5, 1000), (700, 130), (1000, 1100), (64, 3000), (4000, 50)]      # (the first eight: both sides of what a workgroup keeps in LDS)


def check(y, x, steps=5, coef=COEF, eps=1e-7, name=""):
    """y against 64 bits: within the worst-case bound, and within twice what plain fp32 loses (x as the kernel got it)."""
    xd = x.detach().double().cpu(); exact = ns_plain(xd, steps, coef, eps); plain = ns_plain(xd.float(), steps, coef, eps)
    e, ep = rel(y, exact), rel(plain, exact)
    assert e <= HALF[y.dtype] + LOOSE and e <= HALF[y.dtype] + max(2 * ep, 2e-6), (name, tuple(x.shape), e, ep)


@gpu
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("shape", SHAPES)
def test_newton_schulz(shape, dtype):
    x = gradient_like(shape, sum(shape)).to(dtype).cuda()
    keep = x.clone(); y = md().newton_schulz(x)
    assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous() and torch.equal(x, keep)
    check(y, x)


@gpu
@pytest.mark.parametrize("steps", [1, 2, 3, 7, 16])
def test_newton_schulz_steps_and_coefficients(steps):
    x = gradient_like((40, 100), 3).float().cuda()
    check(md().newton_schulz(x, steps=steps, coefficients=(1.875, -1.25, 0.375)), x, steps, (1.875, -1.25, 0.375))
    if steps <= 5:
        check(md().newton_schulz(x, steps=steps), x, steps)


@gpu
def test_newton_schulz_batches_strides_and_views():
    m = md()
    base = gradient_like((3, 2, 70, 90), 5).float().cuda()
    y = m.newton_schulz(base); assert y.shape == base.shape
    for b in range(3):
        for c in range(2):
            assert torch.equal(y[b, c], m.newton_schulz(base[b, c]))              # a matrix does not depend on its batch
    wide = gradient_like((5, 140, 211), 6).float().cuda()
    for v in (wide.transpose(1, 2), wide[:, ::2, ::3], wide[:, 3:100, 1:88], wide[1:4].permute(0, 2, 1)[:, 5:], wide[0], wide[2].t(), wide[:1].expand(3, -1, -1)):
        y = m.newton_schulz(v); assert y.is_contiguous() and torch.equal(y, m.newton_schulz(v.contiguous()))
    flat = torch.empty(33 * 47 + 1, device="cuda", dtype=torch.bfloat16); x = flat[1:].view(33, 47); x.copy_(gradient_like((33, 47), 7))      # 2-byte aligned
    assert torch.equal(m.newton_schulz(x), m.newton_schulz(x.clone()))
    for shape in ((0, 4, 4), (3, 0, 5), (0, 7), (7, 0)):
        assert m.newton_schulz(torch.empty(shape, device="cuda")).shape == shape


@gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e-9, 1.0, 1e18, 1e30])
def test_newton_schulz_extreme_scales_and_the_clamp(scale):
    x = (gradient_like((48, 80), 8, scale=1.0) * scale).float().cuda()
    for eps in (1e-7, 1e-35):                                   # below eps the matrix is not brought to norm 1: its singular values only grow by a^5
        check(md().newton_schulz(x, eps=eps), x, eps=eps, name=eps)


@gpu
def test_newton_schulz_zeros_nan_and_infinities_stay_in_their_matrix():
    m = md(); x = gradient_like((4, 70, 140), 9).float().cuda(); y = m.newton_schulz(x)
    z = x.clone(); z[0] = 0; z[1, 3, 5] = math.nan; z[2, 69, 139] = math.inf
    w = m.newton_schulz(z)
    assert torch.equal(w[0], torch.zeros_like(w[0])) and torch.isnan(w[1]).all() and torch.isnan(w[2]).all() and torch.equal(w[3], y[3])


@gpu
def test_newton_schulz_low_rank():
    """Rank 3 of 40: the 37 null directions hold only what rounding leaves there, amplified by a^5: 1.4e-4 in each of 40 directions, of a result of norm 0.68 sqrt(3) or more."""
    g = torch.Generator().manual_seed(1); x = (torch.randn(40, 3, generator=g, dtype=torch.float64) @ torch.randn(3, 90, generator=g, dtype=torch.float64)).float().cuda()
    assert rel(md().newton_schulz(x), ns_plain(x.double().cpu())) <= 1.4e-4 * math.sqrt(40) / (0.68 * math.sqrt(3))


# ---- the pullback ---------------------------------------------------------------------------------------------------------------
def back_plain(x, dout, steps, coef, eps, dtype):
    x = x.detach().to(dtype).requires_grad_(True); a, b, c = coef
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt().clamp_min(eps)
    y = (x.double() / norm).to(dtype)
    tall = y.shape[-2] > y.shape[-1]
    y = y.transpose(-1, -2) if tall else y
    for _ in range(steps):
        g = y @ y.transpose(-1, -2); y = a * y + (b * g + c * (g @ g)) @ y
    return torch.autograd.grad(y.transpose(-1, -2) if tall else y, x, dout.detach().to(dtype))[0]


def check_back(dx, x, dout, steps=5, coef=COEF, eps=1e-7):
    """The pullback's products carry the same roundings as the iteration's, and G grows by at most about 4 a step as an iterate's singular values by 3.4: the same bounds, with two chains
    (forward, back) of errors instead of one."""
    xd, dd = x.double().cpu(), dout.double().cpu()
    exact, plain = back_plain(xd, dd, steps, coef, eps, torch.float64), back_plain(xd, dd, steps, coef, eps, torch.float32)
    e, ep = rel(dx, exact), rel(plain, exact)
    assert e <= HALF[dx.dtype] + 4 * LOOSE and e <= HALF[dx.dtype] + max(2 * ep, 4e-6), (tuple(x.shape), e, ep)


@gpu
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("shape", [(1, 7), (9, 1), (2, 3), (31, 33), (64, 64), (65, 64), (64, 576), (129, 131), (200, 77), (130, 300), (3, 40, 60), (2, 150, 37), (64, 2000), (20, 3000), (5, 33, 500)])
def test_newton_schulz_pullback(shape, dtype):
    x = gradient_like(shape, sum(shape)).to(dtype).cuda(); d = torch.randn(shape, generator=torch.Generator().manual_seed(2), dtype=torch.float64).to(dtype).cuda()
    keep = x.clone(), d.clone(); dx = md().newton_schulz_pullback(x, d)
    assert dx.shape == x.shape and dx.dtype == dtype and dx.is_contiguous() and torch.equal(x, keep[0]) and torch.equal(d, keep[1])
    check_back(dx, x, d)


@gpu
def test_pullback_against_differences_of_the_forward():
    """<dx, v> against (f(x + h v) - f(x - h v)) / 2h of the kernel's own forward, contracted with dout.  The quotient's error: f's rounding (2e-6 of |y| |dout|) over h, and the third
    derivative's h^2 |v|^3 / |x|^2 term: with h |v| = 1e-3 |x| both are a few 1e-3 of |dout| |y| / |x| |v|; the bound is 1e-2 of that."""
    m = md(); x = gradient_like((24, 40), 11, noise=1.0, scale=1.0).float().cuda(); g = torch.Generator().manual_seed(4)
    d = torch.randn(24, 40, generator=g).cuda(); dx = m.newton_schulz_pullback(x, d, steps=2)
    for _ in range(4):
        v = torch.randn(24, 40, generator=g).cuda(); h = 1e-3 * float(x.norm() / v.norm())
        num = float(((m.newton_schulz(x + h * v, steps=2).double() - m.newton_schulz(x - h * v, steps=2).double()) / (2 * h) * d.double()).sum())
        scale = float(d.norm() * m.newton_schulz(x, steps=2).norm() / x.norm() * v.norm())
        assert abs(num - float((dx.double() * v.double()).sum())) <= 1e-2 * scale


@gpu
@pytest.mark.parametrize("steps", [1, 2, 6])
def test_pullback_steps_strides_and_scales(steps):
    m = md(); co = (1.875, -1.25, 0.375)
    x = gradient_like((2, 90, 41), 12).float().cuda(); d = torch.randn(41, 90, generator=torch.Generator().manual_seed(5)).cuda().t().expand(2, 90, 41)
    check_back(m.newton_schulz_pullback(x, d, steps=steps, coefficients=co), x, d, steps, co)
    for s in (1e-25, 1e20):
        a, b = m.newton_schulz_pullback(x, (d * s), steps=steps, coefficients=co), m.newton_schulz_pullback(x, d, steps=steps, coefficients=co)
        assert rel(a.double() / s, b) <= 1e-6
    assert torch.equal(m.newton_schulz_pullback(x, torch.zeros_like(d), steps=steps), torch.zeros_like(x))


@gpu
def test_pullback_of_a_clamped_and_of_a_zero_matrix():
    """Below eps the normalisation is a division by a constant; at x = 0 that leaves a^steps / eps * dout."""
    m = md(); x = gradient_like((20, 30), 13, scale=1e-9).float().cuda(); d = torch.randn(20, 30, generator=torch.Generator().manual_seed(6)).cuda()
    check_back(m.newton_schulz_pullback(x, d), x, d)
    z = m.newton_schulz_pullback(torch.zeros(20, 30, device="cuda"), d)
    assert rel(z, d.double() * 3.4445 ** 5 / 1e-7) <= 1e-5


@gpu
def test_pullback_nan_stays_in_its_matrix():
    m = md(); x = gradient_like((3, 40, 50), 14).float().cuda(); d = torch.randn(3, 40, 50, generator=torch.Generator().manual_seed(7)).cuda(); dx = m.newton_schulz_pullback(x, d)
    d2, x2 = d.clone(), x.clone(); d2[0, 1, 2] = math.nan; x2[2, 0, 0] = math.inf
    w = m.newton_schulz_pullback(x2, d2)
    assert torch.isnan(w[0]).all() and torch.equal(w[1], dx[1]) and torch.isnan(w[2]).all()


# ---- muon_raw -------------------------------------------------------------------------------------------------------------------
def muon_plain(p, g, m, lr, momentum, nesterov, weight_decay, adjust, grad_scale, steps=5, coef=COEF, eps=1e-7):
    r, c = p.shape[0], p[0].numel(); g = grad_scale * g.double(); m = momentum * m.double() + (1 - momentum) * g
    u = momentum * m + (1 - momentum) * g if nesterov else m
    s = 0.2 * math.sqrt(max(r, c)) if adjust == "rms" else math.sqrt(max(1.0, r / c))
    step = lr * s * ns_plain(u.reshape(r, c), steps, coef, eps).reshape(p.shape)
    return (1 - lr * weight_decay) * p.double() - step, m, step


WEIGHTS = [(64, 3, 3, 3), (37, 53), (1, 700), (129, 65), (300, 1), (1, 1), (16, 16, 1, 1), (96, 8, 3, 3), (255, 257), (64, 63)]


@gpu
@pytest.mark.parametrize("kw", [dict(), dict(nesterov=False, weight_decay=0.1), dict(adjust="rms", momentum=0.0, lr=1e-3), dict(lr=0.0, weight_decay=0.5), dict(grad_scale=-0.125)])
def test_muon_raw(kw):
    """Two steps of odd weights packed with gaps: weights and momenta against 64 bits, the gaps and the gradients as they were.  A weight is off by its own two roundings and the
    orthogonalisation's error times the step."""
    hyper = dict(lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, adjust="spectral", grad_scale=1.0); hyper.update(kw)
    sizes = [int(np.prod(s)) for s in WEIGHTS]; gap = 3; n = sum(sizes) + gap * len(sizes)
    bufs = {k: torch.full((n,), 7.25, device="cuda") for k in "pgm"}; views = {k: [] for k in "pgm"}; at = 0; mask = torch.ones(n, dtype=torch.bool)
    for i, (s, k) in enumerate(zip(WEIGHTS, sizes)):
        for q in "pgm":
            views[q].append(bufs[q][at:at + k].view(s))
        views["p"][-1].copy_(torch.randn(s, generator=torch.Generator().manual_seed(i)) * 0.1)
        for q, off in (("g", 50), ("m", 90)):
            views[q][-1].copy_(gradient_like((s[0], k // s[0]), i + off).reshape(s))
        mask[at:at + k] = False; at += k + gap
    for _ in range(2):
        before = [tuple(views[q][i].double().cpu() for q in "pgm") for i in range(len(WEIGHTS))]; grads = bufs["g"].clone()
        md().muon_raw(views["p"], views["g"], views["m"], **hyper)
        assert torch.equal(bufs["g"], grads)
        for q in "pm":
            assert (bufs[q].cpu()[mask] == 7.25).all()
        for i, (p, g, m) in enumerate(before):
            ep, em, step = muon_plain(p, g, m, **hyper)
            assert float((views["m"][i].double().cpu() - em).abs().max()) <= 3 * 2.0 ** -24 * float(m.abs().max() + g.abs().max() * abs(hyper["grad_scale"]))
            err = (views["p"][i].double().cpu() - ep).norm(); assert float(err) <= float(2 * 2.0 ** -24 * (p.norm() + step.norm()) + 2e-5 * step.norm()), WEIGHTS[i]


@gpu
def test_muon_raw_list_order_and_company():
    """A list in another order gives the same bits.  Alone, a weight may take other tiles (sums in another order): both results are within 2e-5 of the step of the exact one (as above)."""
    m = md(); shapes = [(70, 90), (16, 40), (130, 64), (200, 200)] * 11                  # 44 weights: more than one argument block of the set-up kernel
    def make():
        return [[gradient_like(s, i + 100 * k).float().cuda() for i, s in enumerate(shapes)] for k in range(3)]
    a, b, c = make(), make(), make(); start = [p.clone() for p in a[0]]
    m.muon_raw(*a)
    m.muon_raw(b[0][::-1], b[1][::-1], b[2][::-1])
    assert all(torch.equal(x, y) for k in (0, 2) for x, y in zip(a[k], b[k]))
    for i in range(len(shapes)):
        m.muon_raw([c[0][i]], [c[1][i]], [c[2][i]])
        step = float((a[0][i] - start[i]).norm())
        assert torch.equal(a[2][i], c[2][i]) and float((a[0][i].double() - c[0][i].double()).norm()) <= 4 * 2.0 ** -24 * (float(start[i].norm()) + step) + 4e-5 * step
    small = [[gradient_like((17, 5 + i), i + 100 * k).float().cuda() for i in range(80)] for k in range(3)]; one = [[t.clone() for t in l] for l in small]
    m.muon_raw(*small)                                                                   # 80 weights that fit a workgroup each: three launches
    for i in range(80):
        m.muon_raw([one[0][i]], [one[1][i]], [one[2][i]])
    assert all(torch.equal(x, y) for k in (0, 2) for x, y in zip(small[k], one[k]))
    m.muon_raw([], [], [])
    with pytest.raises(ValueError):
        m.muon_raw([a[0][0].t()], [a[1][0].t()], [a[2][0].t()])
    with pytest.raises(ValueError):
        m.muon_raw([a[0][0][0]], [a[1][0][0]], [a[2][0][0]])
    with pytest.raises(ValueError):
        m.muon_raw([a[0][0]], [a[1][1]], [a[2][0]])
    with pytest.raises(RuntimeError, match="overlaps"):
        m.muon_raw([a[0][0], a[0][0]], [a[1][0], a[1][0]], [a[2][0], a[2][4]])


@gpu
@pytest.mark.parametrize("shape", [(64, 64), (40, 1500), (130, 200), (3, 70, 90), (300, 600), (17, 60, 700), (150, 1000)])
def test_nothing_depends_on_what_the_workspace_held(shape):
    """Rows and columns behind a matrix's last in the workspace may hold anything, NaN too: the same bits after the allocator's memory was filled with NaN and with zeros."""
    m = md(); x = gradient_like(shape, 3).float().cuda(); d = torch.randn(shape, generator=torch.Generator().manual_seed(4)).cuda(); got = []
    for fill in (math.nan, 0.0):
        out = []
        for f in (lambda: m.newton_schulz(x), lambda: m.newton_schulz_pullback(x, d)):
            torch.cuda.empty_cache(); junk = torch.full((1 << 27,), fill, device="cuda"); torch.cuda.synchronize(); del junk      # 512 MB: the next workspace is cut from it
            out.append(f())
        p, mo = x.reshape(-1, shape[-1]).clone(), torch.zeros(x.numel() // shape[-1], shape[-1], device="cuda"); junk = torch.full((1 << 27,), fill, device="cuda"); del junk
        m.muon_raw([p], [x.reshape(-1, shape[-1])], [mo]); got.append(out + [p, mo])
    assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(*got))


# ---- streams, graphs, repeatability ---------------------------------------------------------------------------------------------------
@gpu
def test_side_streams_and_two_calls_at_once():
    m = md(); xs = [gradient_like((200, 500), i).float().cuda() for i in range(2)]; want = [m.newton_schulz(x) for x in xs]; back = m.newton_schulz_pullback(xs[0], xs[1]); torch.cuda.synchronize()
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for s, x in zip(st, xs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(m.newton_schulz(x)); got.append(m.newton_schulz_pullback(xs[0], xs[1]))
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[1]) and torch.equal(got[1], back) and torch.equal(got[3], back)


@gpu
def test_captured_and_replayed():
    """newton_schulz, its pullback and a Muon step in graphs, replayed between eager calls on other data; two graphs of one pool."""
    m = md(); x = gradient_like((2, 90, 150), 20).float().cuda(); d = torch.randn(2, 90, 150, generator=torch.Generator().manual_seed(8)).cuda()
    p, g, mo = [gradient_like((90, 300), 21 + i).float().cuda() for i in range(3)]
    m.newton_schulz(x); torch.cuda.synchronize()
    g1 = torch.cuda.CUDAGraph(); g2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        y, dx = m.newton_schulz(x), m.newton_schulz_pullback(x, d)
    with torch.cuda.graph(g2, pool=g1.pool()):
        m.muon_raw([p], [g], [mo])
    for r in range(4):
        x.copy_(gradient_like((2, 90, 150), 30 + r)); p0, m0 = p.clone(), mo.clone()
        g1.replay(); torch.cuda.synchronize()
        assert torch.equal(y, m.newton_schulz(x)) and torch.equal(dx, m.newton_schulz_pullback(x, d))
        g2.replay(); torch.cuda.synchronize()
        m.muon_raw([p0], [g], [m0]); assert torch.equal(p, p0) and torch.equal(mo, m0)


@gpu
def test_orthogonalised_weight_trains_through_its_pullback():
    """A run of the operators together: w = newton_schulz(v), loss 1/2 |w - target|^2, dv by the pullback, v stepped by muon_raw; every step's gradient against 64 bits."""
    m = md(); v = gradient_like((48, 96), 40, noise=1.0, scale=1.0).float().cuda(); t = m.newton_schulz(gradient_like((48, 96), 41, noise=1.0).float().cuda()); mo = torch.zeros_like(v)
    for _ in range(3):
        w = m.newton_schulz(v); dv = m.newton_schulz_pullback(v, w - t)
        check(w, v); check_back(dv, v, w - t)
        m.muon_raw([v], [dv], [mo], lr=0.05)


# ---- the model's own path -------------------------------------------------------------------------------------------------------------
def make_model(depth=18, N=2, C=1, H=64, W=96, seed=3, lr=1e-4):
    m = md(); syn = md2amd.synthetic; K, iK = syn.depth10k_intrinsics(W, H)
    params = m.Params(target_size=(W, H), batch_size=N, automasking=False)
    cache = m.TrainCache(m.SSIM(), m.Backproject(W, H), m.Project(W, H), K, iK, 2, [1, 3], [0.125, 0.25, 0.5, 1.0])
    enc = m.ResidualNetwork(depth, in_channels=C); model = m.Model(enc, m.DepthDecoder(list(enc.stages), [2, 3, 4, 5]), m.PoseDecoder(enc.stages[-1]), lr=lr)
    model.load_params(syn.init_params(C, seed=seed, randomize_affine=True, depth=depth))
    return model, params, cache, torch.from_numpy(syn.synthetic_triplets(N, C, H, W, seed=5)).cuda()


def arrays(flat, depth=18):
    out, off = {}, 0
    for name, kind, shape in md2amd.synthetic.param_layout(1, depth):
        n = int(np.prod(shape)); out[name] = (kind, flat[off:off + n].reshape(shape)); off += n
    return out


def hidden(name, kind):
    return kind == "W" and name != "enc.stem.W" and not name.startswith("dec.head") and name != "pose.pose3.W"


@gpu
@pytest.mark.parametrize("depth", [18, 50])
def test_model_update_with_muon(depth):
    """Two steps of update(Muon, model) against 64 bits from the model's own gradients: the hidden convolutions as matrices, everything else exactly as an ADAM step leaves it."""
    m = md(); a, params, cache, x = make_model(depth); b = make_model(depth)[0]
    opt = m.Muon(eta=1e-3, weight_decay=0.1, adjust="rms", adam_eta=2e-4); mom = None
    for _ in range(2):
        m.train_step(a, x, None, cache, params, do_update=False); m.train_step(b, x, None, cache, params, do_update=False)
        p0, g = a.params(), a.grads(); b.param_buffer().copy_(a.param_buffer()); b.grad_buffer().copy_(a.grad_buffer())
        m.update(opt, a, grad_scale=0.5); m.update(m.ADAM(2e-4), b, grad_scale=0.5)
        p1, q1 = arrays(a.params(), depth), arrays(b.params(), depth); p0, g = arrays(p0, depth), arrays(g, depth); got = arrays(a.muon_state(), depth)
        mom = mom or {k: np.zeros_like(v) for k, (_, v) in p0.items()}; count = 0
        for name, (kind, after) in p1.items():
            if not hidden(name, kind):
                assert np.array_equal(after, q1[name][1]), name
                assert not got[name][1].any(), name
                continue
            count += 1; t = [torch.from_numpy(np.ascontiguousarray(v)) for v in (p0[name][1], g[name][1], mom[name])]
            if t[0].numel() > 1 << 20 and depth == 50:            # (the largest ones: their rows' norms only, to keep the test short)
                assert np.isfinite(after).all() and not np.array_equal(after, p0[name][1]); mom[name] = got[name][1]; continue
            ep, em, step = muon_plain(*t, 1e-3, 0.95, True, 0.1, "rms", 0.5)
            assert float((torch.from_numpy(np.ascontiguousarray(got[name][1])).double() - em).abs().max()) <= 3 * 2.0 ** -24 * float(t[1].abs().max() + t[2].abs().max()), name
            assert float((torch.from_numpy(np.ascontiguousarray(after)).double() - ep).norm()) <= float(2 * 2.0 ** -24 * (t[0].double().norm() + step.norm()) + 2e-5 * step.norm()), name
            mom[name] = got[name][1]
        assert count == {18: 32, 50: 65}[depth]


@gpu
def test_a_muon_handle_refuses_adam_until_its_state_is_dropped():
    m = md(); model, params, cache, x = make_model(); L = md2amd._lib.lib()
    with pytest.raises(RuntimeError, match="no device handle"):
        m.update(m.Muon(), model)
    m.train_step(model, x, None, cache, params); assert model.muon_state() is None
    for bad in (dict(eta=-1.0), dict(momentum=1.0), dict(weight_decay=-1.0), dict(steps=0), dict(eps=0.0), dict(coefficients=(9.0, 0.0, 0.0))):
        with pytest.raises(RuntimeError, match="muon_step"):
            m.update(m.Muon(**bad), model)
    with pytest.raises(ValueError):
        m.update(m.Muon(adjust="x"), model)
    assert model.muon_state() is None                                     # a refused call leaves the handle ADAM's
    m.update(m.Muon(), model); p = model.params(); assert np.abs(model.muon_state()).max() > 0
    with pytest.raises(RuntimeError, match="stepped by Muon"):
        m.update(m.ADAM(1e-4), model)
    with pytest.raises(RuntimeError, match="stepped by Muon"):
        m.train_step(model, x, None, cache, params)
    assert np.array_equal(model.params(), p)
    assert L.md2_muon_state_set(model._h, p.ctypes.data_as(ctypes.c_void_p), 7) == 2 and L.md2_muon_state_set(model._h, None, 7) == 2
    model.load_params(p); assert model.muon_state() is None                # new parameters: the optimiser starts anew
    m.update(m.Muon(), model); p = model.params(); model.load_muon_state(None); st = model._opt_and_bn_state()
    assert model.muon_state() is None and not st[0].any() and not st[1].any() and st[2:4] == (1.0, 1.0)
    m.train_step(model, x, None, cache, params); assert not np.array_equal(model.params(), p)


@gpu
def test_muon_state_survives_a_handle_rebuild_and_a_checkpoint(tmp_path):
    m = md(); model, params, cache, x = make_model(); opt = m.Muon(eta=1e-3)
    for _ in range(2):
        m.train_step(model, x, None, cache, params, do_update=False); m.update(opt, model)
    st, adam = model.muon_state(), model._opt_and_bn_state()
    m.save_checkpoint(model, str(tmp_path / "c.npz"))
    m.train_loss(model, x[:1].contiguous(), None, cache, m.Params(target_size=(96, 64), batch_size=1, automasking=False))      # another batch size: a new handle
    assert np.array_equal(model.muon_state(), st) and np.array_equal(model._opt_and_bn_state()[0], adam[0])
    other, _, _, _ = make_model(seed=9); m.train_step(other, x, None, cache, params, do_update=False); m.load_checkpoint(other, str(tmp_path / "c.npz"))
    assert np.array_equal(other.muon_state(), st) and np.array_equal(other._opt_and_bn_state()[1], adam[1]) and other._opt_and_bn_state()[2] == adam[2]
    plain, _, _, _ = make_model(seed=9); m.train_step(plain, x, None, cache, params); m.save_checkpoint(plain, str(tmp_path / "d.npz"))
    m.load_checkpoint(other, str(tmp_path / "d.npz")); assert other.muon_state() is None and np.array_equal(other._opt_and_bn_state()[0], plain._opt_and_bn_state()[0])


@gpu
def test_muon_step_beside_the_training_step_and_in_one_process_data_parallel():
    """Training steps with Muon, the two-stream step around it, equal one after the other and through DataParallel (one rank)."""
    m = md(); opt = m.Muon(eta=1e-3); m.set_deterministic(True)
    try:
        runs = []
        for way in range(2):
            model, params, cache, x = make_model(); dp = md2amd.parallel.DataParallel(model, comm="torch"); losses = []
            for _ in range(3):
                if way:
                    losses.append(float(dp.train_step(x, None, cache, params, optimizer=opt)))
                else:
                    loss = m.train_loss(model, x, None, cache, params)[0]; m.gradient(model); m.update(opt, model); losses.append(float(loss))
            runs.append((losses, model.params(), model.muon_state()))
        assert runs[0][0] == runs[1][0] and np.array_equal(runs[0][1], runs[1][1]) and np.array_equal(runs[0][2], runs[1][2]) and all(np.isfinite(runs[0][0]))
    finally:
        m.set_deterministic(False)


@gpu
def test_train_takes_the_optimizer(tmp_path):
    class Frames:                                                         # what train() reads of a dataset
        resolution, target_id, source_ids = (96, 64), 2, (1, 3); K, invK = md2amd.synthetic.depth10k_intrinsics(96, 64)
        x = md2amd.synthetic.synthetic_triplets(4, 1, 64, 96, seed=7)
        def __len__(self): return 4
        def __getitem__(self, i): return self.x[i]
    model, losses = md2amd.train.train([Frames()], str(tmp_path / "l"), str(tmp_path / "s"), batch_size=2, n_epochs=2, log_iter=100, save_iter=2, quiet=True, optimizer=md().Muon(eta=1e-3, adam_eta=5e-5))
    assert len(losses) == 4 and np.isfinite(losses).all() and model.lr == 5e-5 and np.abs(model.muon_state()).max() > 0
    assert any("muon_m" in np.load(f) for f in (tmp_path / "s").glob("*.npz"))


# ---- arguments at the ends of their ranges ----------------------------------------------------------------------------------------------
def test_an_eps_past_the_largest_float_is_refused():
    for eps in (3.5e38, 1e308):
        assert ns_c(eps=eps) == 2 and "eps" in last_error()
        assert muon_c(eps=eps) == 2 and "eps" in last_error()
    assert ns_c(eps=3.4e38) == 2 and "workspace" in last_error()


@gpu
@pytest.mark.parametrize("shape", [(48, 80), (90, 150)])
def test_the_smallest_and_largest_eps(shape):
    """Zeros over an eps whose reciprocal no double holds are zeros; a matrix far below a huge eps is only scaled and grown."""
    m = md()
    assert torch.equal(m.newton_schulz(torch.zeros(shape, device="cuda"), eps=1e-320), torch.zeros(shape, device="cuda"))
    x = gradient_like(shape, 8, scale=1.0)
    check(m.newton_schulz(x.float().cuda(), eps=1e-320), x.float())
    check(m.newton_schulz(x.float().cuda(), eps=1e30), x.float(), eps=1e30)
    check(m.newton_schulz((x * 1e30).float().cuda(), eps=1e38), (x * 1e30).float(), eps=1e38)


@gpu
@pytest.mark.parametrize("shape", [(24, 40), (70, 90), (130, 200)])
@pytest.mark.parametrize("coef", [(1.0, 0.0, 0.0), (1.5, -0.5, 0.0), (0.75, 0.0, -0.25), (0.0, 1.0, 0.0), (0.0, 0.0, 0.0)])
def test_coefficients_that_are_zero(shape, coef):
    m = md(); x = gradient_like(shape, 14, noise=1.0).float().cuda(); d = torch.randn(shape, generator=torch.Generator().manual_seed(9)).cuda()
    y, dx = m.newton_schulz(x, steps=1, coefficients=coef), m.newton_schulz_pullback(x, d, steps=1, coefficients=coef)
    if not any(coef):
        assert not y.any() and not dx.any()
        return
    check(y, x, 1, coef); check_back(dx, x, d, 1, coef)
    if coef[0]:
        check(m.newton_schulz(x, steps=3, coefficients=coef), x, 3, coef); check_back(m.newton_schulz_pullback(x, d, steps=3, coefficients=coef), x, d, 3, coef)


@pytest.mark.parametrize("kw,refused", [(dict(y=4096), True), (dict(y=4096 + 252), True), (dict(y=4096 - 252), True), (dict(y=4096 + 256), False), (dict(y=4096 - 256), False),
                                        (dict(batch=2, strides=(1024, 8, 1), y=4096 + 2048), True), (dict(batch=2, strides=(0, 0, 0), y=4096 + 4), False), (dict(strides=(1 << 62, 1 << 62, 1 << 62)), True)])
def test_a_result_that_overlaps_an_input_is_refused(kw, refused):
    """8 x 8 fp32 matrices of 256 bytes at 4096 (a call that is not refused for it is for its workspace)."""
    assert ns_c(**kw) == 2 and ("overlaps" if refused else "workspace") in last_error(), last_error()
    if set(kw) == {"y"}:
        L = md2amd._lib.lib(); st = (ctypes.c_int64 * 3)(64, 8, 1); co = (ctypes.c_double * 3)(*COEF)
        assert L.md2_newton_schulz_bwd(65536, 4096, kw["y"], 1, 8, 8, st, st, 0, 5, co, 1e-7, 4096, 0, None) == 2 and ("overlaps" if refused else "workspace") in last_error()


@gpu
def test_a_model_step_cannot_be_captured():
    """The ADAM part's bias corrections are arguments of its launch: a replayed step would repeat them, so the call is refused and nothing is recorded or changed."""
    m = md(); model, params, cache, x = make_model(); m.train_step(model, x, None, cache, params, do_update=False); p = model.params()
    for first in (True, False):
        side = torch.zeros(4, device="cuda"); torch.cuda.synchronize(); graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            side.add_(1)
            with pytest.raises(RuntimeError, match="captured"):
                m.update(m.Muon(), model)
        graph.replay(); torch.cuda.synchronize()
        assert (side == 1).all() and np.array_equal(model.params(), p) and (model.muon_state() is None) == first
        m.update(m.Muon(), model); q = model.params(); assert not np.array_equal(p, q); p = q


def test_more_work_than_a_launch_can_hold_is_refused():
    """(such a call's workspace would be 16 TB and more)"""
    L = md2amd._lib.lib()
    assert L.md2_newton_schulz_workspace(1 << 20, 1000, 2000, 5, 0) == -1 and L.md2_newton_schulz_workspace(1 << 20, 100, 200, 5, 0) > 0


# ---- ranges of the numbers inside --------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("shape", [(1, 1), (20, 30), (70, 90), (200, 130)])
@pytest.mark.parametrize("coef,steps", [((1.0, -1.0, 0.0), 2), ((0.75, 0.0, -0.25), 3), ((0.5, 0.0, 0.0), 6)])
def test_pullback_of_a_clamped_matrix_with_coefficients_that_shrink(shape, coef, steps):
    """A matrix below eps is carried larger; where the coefficients let singular values shrink, an iterate must not be carried past the bound by which G X^T is scaled (its pairs would be
    infinite, the next product NaN).  One entry holds nearly all of x and dout, so that entries come as near to the norms' bounds as they can."""
    g = torch.Generator().manual_seed(3); z = 1e-3 * torch.randn(shape, generator=g, dtype=torch.float64) / max(shape); z[shape[0] // 2, shape[1] // 3] = 1.0; z /= z.norm()
    for r in (0.01, 0.03, 0.06, 0.1, 0.2, 0.3, 0.45, 0.7):
        x, d = (z * r * 1e-7).float().cuda(), z.float().cuda()
        check_back(md().newton_schulz_pullback(x, d, steps=steps, coefficients=coef), x, d, steps, coef)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(3, 5), (70, 90)])
def test_pullback_of_the_smallest_and_largest_gradients(shape, dtype):
    """dx = (dout - X0 <X0, dout>) / |x| for coefficients (1, 0, 0).  Powers of two scale x and dout until |dout| / |x| is subnormal times 2^14: the normal dx has the bits of the unscaled
    call's, moved by the exponent.  Where dx passes fp32's range it is infinite, and its zeros stay zeros."""
    m = md(); x = gradient_like(shape, 51, noise=1.0, scale=1.0); x[0, 0] = 9 * x.norm(); d = torch.randn(shape, generator=torch.Generator().manual_seed(52), dtype=torch.float64)
    x, d = (x / x.norm()).to(dtype).cuda(), d.to(dtype).cuda(); ref = m.newton_schulz_pullback(x, d, steps=1, coefficients=(1.0, 0.0, 0.0)).double()
    for sx, sd in ((2.0 ** 60, 2.0 ** -63), (2.0 ** 30, 2.0 ** -94), (2.0 ** 62, 2.0 ** -60), (2.0 ** -40, 2.0 ** 80)):
        got = m.newton_schulz_pullback(x * sx, d * sd, steps=1, coefficients=(1.0, 0.0, 0.0), eps=1e-30).double(); want = ref * (sd / sx); normal = want.abs() >= 2.0 ** -125
        assert normal.sum() >= want.numel() // 4 and torch.equal(got[normal], want[normal]), (sx, sd)
    for eps in (1e-12, 1e-320):                                  # a^5 / eps dout, past 3.4e38 everywhere but where dout is 0
        z = d * 1e30; z[1:] = 0; got = m.newton_schulz_pullback(torch.zeros_like(x), z, eps=eps)
        assert torch.equal(got[0], torch.copysign(torch.full_like(z[0], math.inf), z[0])) and not got[1:].any()


@gpu
@pytest.mark.parametrize("momentum", [0.9999, 1 - 1e-7, 1 - 1e-8])
@pytest.mark.parametrize("shape", [(24, 40), (70, 90)])
def test_a_momentum_next_to_one(shape, momentum):
    """From zero, m = (1 - momentum) g: three roundings (1 - momentum, grad_scale g, their product), however near 1 the momentum is.  The direction does not depend on the size of u."""
    p, g, mo = torch.zeros(shape, device="cuda"), gradient_like(shape, 61, noise=1.0, scale=1.0).float().cuda(), torch.zeros(shape, device="cuda")
    md().muon_raw([p], [g], [mo], lr=1.0, momentum=momentum, nesterov=False, grad_scale=0.75, eps=1e-30)
    want = (1 - momentum) * 0.75 * g.double()
    assert float(((mo.double() - want).abs() / want.abs()).max()) <= 4 * 2.0 ** -24
    check(-p, want.float(), eps=1e-30)


@pytest.mark.parametrize("kw,word", [(dict(lr=1e39), "shape factor"), (dict(lr=2e38, rows=(64,), cols=(1,), p=(4096,), g=(8192,), m=(16384,)), "shape factor"), (dict(lr=1e20, decay=1e19), "weight_decay"),
                                     (dict(lr=3e38), "workspace"), (dict(lr=1e19, decay=1e19), "workspace")])
def test_a_learning_rate_that_no_float_holds_is_refused(kw, word):
    """(as infinite factors they would make NaN of weights whose update is zero)"""
    assert muon_c(**kw) == 2 and word in last_error(), last_error()


@gpu
def test_a_model_step_refuses_such_a_learning_rate_and_stays_adams():
    m = md(); model, params, cache, x = make_model(); m.train_step(model, x, None, cache, params); p = model.params()
    for kw in (dict(eta=1e38, adjust="rms"), dict(eta=1e20, weight_decay=1e19)):
        with pytest.raises(RuntimeError, match="range"):
            m.update(m.Muon(**kw), model)
    assert model.muon_state() is None and np.array_equal(model.params(), p)
    m.train_step(model, x, None, cache, params); assert not np.array_equal(model.params(), p)


# ---- a refused update changes nothing ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("which", ["muon", "adam"])
def test_a_refused_update_keeps_the_models_step_size(monkeypatch, which):
    """The library's part is a stand-in that refuses the step, or the step size itself: model.lr and the handle's step size are what they were; an accepted step keeps the new one."""
    import contextlib
    m = md(); calls = []; answer = {"step": 2, "lr": 0}
    class Lib:
        def md2_set_lr(self, h, v): calls.append(v); return answer["lr"] if v < 0 else 0
        def md2_set_stream(self, h, s): return 0
        def md2_muon_step(self, *a): return answer["step"]
        def md2_adam_step(self, *a): return answer["step"]
        def md2_last_error(self, h): return b"refused"
    monkeypatch.setattr(m._lib, "lib", lambda: Lib()); monkeypatch.setattr(m, "_stream", lambda: None); monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    model = m.Model.__new__(m.Model); model._lr, model._h, model._shape = 1e-4, 1, (0,)
    step = (lambda eta: m.update(m.Muon(adam_eta=eta), model)) if which == "muon" else (lambda eta: m.update(m.ADAM(eta), model))
    try:
        with pytest.raises(RuntimeError, match="refused"):
            step(3e-3)
        assert model.lr == 1e-4 and (not calls or calls[-1] == 1e-4)
        answer["lr"] = 2
        with pytest.raises(RuntimeError, match="refused"):
            step(-1.0)
        assert model.lr == 1e-4
        answer["step"] = 0; step(2e-3); assert model.lr == 2e-3 and calls[-1] == 2e-3
    finally:
        model._h = None


@gpu
def test_a_refused_step_keeps_the_handles_step_size():
    m = md(); model, params, cache, x = make_model(); other = make_model()[0]
    for mm in (model, other):
        m.train_step(mm, x, None, cache, params, do_update=False)
    for bad in (dict(eta=-1.0), dict(momentum=1.0), dict(steps=0), dict(coefficients=(9.0, 0.0, 0.0)), dict(adam_eta=-1.0)):
        with pytest.raises(RuntimeError):
            m.update(m.Muon(**{"adam_eta": 0.5, **bad}), model)
    assert model.lr == 1e-4 and model.muon_state() is None
    other.grad_buffer().copy_(model.grad_buffer()); other.param_buffer().copy_(model.param_buffer())
    for mm in (model, other):
        m.update(None, mm)
    assert np.array_equal(model.params(), other.params())
    m.update(m.Muon(adam_eta=2e-4), model)
    with pytest.raises(RuntimeError, match="stepped by Muon"):
        m.update(m.ADAM(0.5), model)
    assert model.lr == 2e-4


# ---- the state's exchange between ranks ------------------------------------------------------------------------------------------------------
@gpu
def test_broadcast_state_leaves_no_rank_waiting_for_one_without_memory():
    """One rank's part of md2_broadcast_state against a stand-in for RCCL: whether every rank can hold the momentum is agreed on (a reduction that each takes part in) before any of them enters
    its broadcast, and where one cannot, none does, all return an error, and a momentum allocated for it is given back.  The failing allocation is the host's: nothing reaches the device."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__)); assert os.path.exists(os.path.join(here, "native", "libfake_rccl.so")), "run __graft_entry__.build()"
    r = subprocess.run([sys.executable, "-u", os.path.join(here, "fake_rccl_child.py")], capture_output=True, text=True, timeout=100); assert r.returncode == 0, r.stdout + r.stderr
    got = {l.split()[0]: l.split(maxsplit=6)[1:] for l in r.stdout.splitlines() if l.split() and l.split()[0] in ("nobody", "dropped", "given", "kept", "other_cannot", "other_cannot_kept", "cannot")}
    #                            status, broadcasts (parameters, two moments, statistics, the three numbers; the momentum), reductions, this rank's answer, has Muon state
    assert {k: tuple(float(q) for q in v[:5]) for k, v in got.items()} == {
        "nobody": (0, 5, 0, -1, 0), "dropped": (0, 5, 0, -1, 0), "given": (0, 6, 1, 1, 1), "kept": (0, 6, 1, 1, 1),
        "other_cannot": (3, 5, 1, 1, 0), "other_cannot_kept": (3, 5, 1, 1, 1), "cannot": (3, 5, 1, 0, 0)}, r.stdout
    assert "another rank" in got["other_cannot"][5] and "no device memory" in got["cannot"][5]


@gpu
def test_muon_through_the_librarys_own_communicator():
    """A handle with Muon state joins a communicator (of one rank: RCCL takes no two on a card): its momentum comes through md2_broadcast_state unchanged, and steps with the gradients summed by
    the library equal steps without a communicator, bit for bit."""
    m = md(); opt = m.Muon(eta=1e-3); m.set_deterministic(True)
    try:
        runs = []
        for comm in ("torch", "rccl"):
            model, params, cache, x = make_model()
            for _ in range(2):
                m.train_step(model, x, None, cache, params, do_update=False); m.update(opt, model)
            st = model.muon_state(); dp = md2amd.parallel.DataParallel(model, comm=comm, x_like=x, parameters=params, cache=cache)
            assert np.array_equal(model.muon_state(), st) and st.any()
            losses = [float(dp.train_step(x, None, cache, params, optimizer=opt)) for _ in range(2)]
            runs.append((losses, model.params(), model.muon_state(), model._opt_and_bn_state()[:4])); model.close()
        assert runs[0][0] == runs[1][0] and all(np.array_equal(a, b) for a, b in zip(runs[0][1:3], runs[1][1:3])) and all(np.array_equal(a, b) for a, b in zip(runs[0][3], runs[1][3]))
    finally:
        m.set_deterministic(False)


# ---- 128-tiles ---------------------------------------------------------------------------------------------------------------------------------
def tiles(shape, pullback, steps=5):
    """-> (tile sides, whether the K axis is cut) of X X^T, b A + c A A, S, V and the products with the matrix."""
    b, r, c = shape; I = ctypes.c_int32 * 5; side, pieces = I(), I()
    assert md2amd._lib.lib().md2_newton_schulz_tiles(b, r, c, steps, pullback, side, pieces) == 0
    return tuple(side), tuple(int(p > 1) for p in pieces)


def test_which_kernels_a_call_takes():
    L = md2amd._lib.lib(); I = ctypes.c_int32 * 5
    assert tiles((1, 64, 576), 0) == ((0,) * 5, (0,) * 5) and tiles((1, 64, 576), 1)[0][1::2] == (0, 0)      # one launch | B and V by the workgroups of A and S
    assert tiles((3, 4601, 509), 1) == tiles((3, 509, 4601), 1)
    assert L.md2_newton_schulz_tiles(0, 4, 4, 5, 0, I(), I()) == 2 and L.md2_newton_schulz_tiles(1, 4, 4, 0, 0, I(), I()) == 2 and L.md2_newton_schulz_tiles(1, 4, 4, 5, 0, None, I()) == 2


def held(e, ep, dtype, loose, floor):
    assert e <= HALF[dtype] + loose and e <= HALF[dtype] + max(2 * ep, floor), (e, ep)


def on_the_gpu(x, f):
    """f of every matrix of the batch by itself, in 64 bits and in 32, where x is."""
    return tuple(torch.stack([f(i, t) for i in range(x.shape[0])]) for t in (torch.float64, torch.float32))


# (batch, rows, columns), its tile sides and which K axes are cut: one of the smallest for each combination with a 128-tile in it that sizes of up to 1500 and batches of up to 24 have
FORWARD_128 = [((6, 129, 903), (64, 64, 0, 0, 128), (0, 0, 0, 0, 0)), ((1, 509, 4601), (64, 64, 0, 0, 128), (1, 0, 0, 0, 0)), ((1, 4608, 512), (64, 64, 0, 0, 128), (1, 0, 0, 0, 0)),
               ((24, 257, 335), (64, 128, 0, 0, 128), (0, 0, 0, 0, 0)), ((1, 997, 4501), (128, 64, 0, 0, 128), (1, 0, 0, 0, 0)), ((2, 997, 997), (128, 128, 0, 0, 64), (1, 1, 0, 0, 0)),
               ((24, 257, 257), (128, 128, 0, 0, 128), (0, 0, 0, 0, 0)), ((8, 1283, 641), (128, 128, 0, 0, 128), (1, 0, 0, 0, 0)), ((2, 997, 1297), (128, 128, 0, 0, 128), (1, 1, 0, 0, 0))]
BACK_128 = [((12, 129, 465), (64, 64, 64, 64, 128), (0, 0, 0, 0, 0)), ((6, 903, 129), (64, 64, 64, 64, 128), (0, 0, 1, 0, 0)), ((1, 512, 4608), (64, 64, 64, 64, 128), (1, 0, 1, 1, 0)),
            ((12, 197, 1379), (64, 64, 128, 64, 128), (0, 0, 1, 0, 0)), ((1, 997, 1995), (64, 64, 128, 64, 64), (0, 0, 1, 0, 0)), ((4, 641, 641), (64, 64, 128, 128, 64), (0, 0, 1, 1, 0)),
            ((4, 833, 641), (64, 64, 128, 128, 128), (0, 0, 1, 1, 0)), ((24, 257, 335), (64, 128, 64, 64, 128), (0, 0, 0, 0, 0)), ((1, 1000, 4500), (128, 64, 128, 64, 128), (1, 0, 1, 0, 0)),
            ((4, 641, 1283), (128, 64, 128, 128, 64), (1, 0, 1, 1, 0)), ((3, 1539, 769), (128, 64, 128, 128, 128), (1, 0, 1, 1, 0)), ((24, 257, 257), (128, 128, 64, 64, 128), (0, 0, 0, 0, 0)),
            ((2, 997, 997), (128, 128, 128, 128, 64), (1, 1, 1, 1, 0)), ((24, 385, 385), (128, 128, 128, 128, 128), (0, 0, 0, 0, 0)), ((2, 997, 1297), (128, 128, 128, 128, 128), (1, 1, 1, 1, 0))]


def test_the_128_tile_cases_take_128_tiles():
    for cases, pullback in ((FORWARD_128, 0), (BACK_128, 1)):
        for shape, side, cut in cases:
            assert tiles(shape, pullback) == (side, cut), shape


@gpu
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("shape", [c[0] for c in FORWARD_128])
def test_newton_schulz_in_128_tiles(shape, dtype):
    x = gradient_like(shape, sum(shape)).to(dtype).cuda(); y = md().newton_schulz(x)
    exact, plain = on_the_gpu(x, lambda i, t: ns_plain(x[i].to(t)))
    held(rel(y, exact), rel(plain, exact), dtype, LOOSE, 2e-6)


@gpu
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("shape", [c[0] for c in BACK_128])
def test_newton_schulz_pullback_in_128_tiles(shape, dtype):
    x = gradient_like(shape, sum(shape)).to(dtype).cuda(); d = torch.randn(shape, generator=torch.Generator().manual_seed(2), dtype=torch.float64).to(dtype).cuda()
    dx = md().newton_schulz_pullback(x, d)
    exact, plain = on_the_gpu(x, lambda i, t: back_plain(x[i], d[i], 5, COEF, 1e-7, t))
    held(rel(dx, exact), rel(plain, exact), dtype, 4 * LOOSE, 4e-6)


@gpu
@pytest.mark.parametrize("shape,pullback", [((8, 641, 641), 1), ((2, 997, 1297), 1), ((1, 509, 4601), 1), ((24, 257, 335), 0)])
def test_128_tiles_do_not_depend_on_what_the_workspace_held(shape, pullback):
    m = md(); x = gradient_like(shape, 3).float().cuda(); d = torch.randn(shape, generator=torch.Generator().manual_seed(4)).cuda(); got = []
    assert tiles(shape, pullback)[0][4] == 128
    for fill in (math.nan, 0.0):
        torch.cuda.empty_cache(); junk = torch.full((1 << 28,), fill, device="cuda"); torch.cuda.synchronize(); del junk      # 1 GB: the workspace is cut from it
        got.append(m.newton_schulz_pullback(x, d) if pullback else m.newton_schulz(x))
    assert torch.equal(*got) and torch.isfinite(got[0]).all()


@gpu
def test_the_largest_weights_of_the_resnet50_network():
    """test_model_update_with_muon leaves the values of ResNet-50's weights of more than 2^20 elements unchecked (256 x 18432, 256 x 11520, 2048 x 1024, 512 x 4608, ...: 128-tiles and cut K axes of
    a list).  Here they are held to the same bounds, against 64 bits where the card multiplies: the momentum element by element, the weight by its step."""
    m = md(); model, params, cache, x = make_model(50); opt = m.Muon(eta=1e-3, weight_decay=0.1, adjust="rms"); mom = None
    for _ in range(2):
        m.train_step(model, x, None, cache, params, do_update=False); p0, g = arrays(model.params(), 50), arrays(model.grads(), 50)
        m.update(opt, model, grad_scale=0.5); p1, got = arrays(model.params(), 50), arrays(model.muon_state(), 50); count = 0
        for name, (kind, after) in p1.items():
            if not hidden(name, kind) or after.size <= 1 << 20:
                continue
            count += 1; up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
            t = up(p0[name][1]), up(g[name][1]), up(mom[name][1]) if mom else torch.zeros(after.shape, device="cuda")
            ep, em, step = muon_plain(*t, 1e-3, 0.95, True, 0.1, "rms", 0.5); a, mu = up(after).double(), up(got[name][1]).double()
            assert float((mu - em).abs().max()) <= 3 * 2.0 ** -24 * float(t[1].abs().max() + t[2].abs().max()), name
            assert float((a - ep).norm()) <= float(2 * 2.0 ** -24 * (t[0].double().norm() + step.norm()) + 2e-5 * step.norm()), name
        assert count == 7
        mom = got


@gpu
def test_adams_bits_do_not_depend_on_which_kernel_steps_a_parameter():
    """adam_raw on an aligned buffer (four parameters a thread, the last ones singly) and on one that begins 4 bytes later (all singly); the listed ranges that Muon leaves to ADAM are held to the
    plain ADAM step, bit for bit, in test_model_update_with_muon."""
    m = md(); n = 4099; g = torch.Generator().manual_seed(71); start = [torch.randn(n, generator=g) * s for s in (0.1, 1e-3, 1e-3)] + [torch.rand(n, generator=g) * 1e-6]; got = []
    for off in (0, 1):
        t = [torch.zeros(n + 4, device="cuda")[off:off + n] for _ in range(4)]
        for a, b in zip(t, start):
            a.copy_(b)
        for step in (1, 2, 3):
            m.adam_raw(*t, step, lr=1e-3, grad_scale=0.5)
        got.append([a.clone() for a in t])
    assert all(torch.equal(a, b) for a, b in zip(*got)) and not torch.equal(got[0][0].cpu(), start[0])
    # the moments' roundings: m = fma(0.9, m, 0.1 g), v = fma(g, 0.001 g, 0.999 v) (in 64 bits, which hold the fused product; two roundings of a sum differ from one in 2^-29 of cases)
    f = np.float32; b1, b2 = f(0.9), f(0.999); m0, v0, ge = start[2].numpy(), start[3].numpy(), start[1].numpy() * f(0.5)
    for _ in range(3):
        m0 = (np.float64(b1) * m0 + np.float64((f(1) - b1) * ge)).astype(f); v0 = (np.float64(ge) * ((f(1) - b2) * ge) + np.float64(b2 * v0)).astype(f)
    assert (got[0][2].cpu().numpy() != m0).sum() <= 2 and (got[0][3].cpu().numpy() != v0).sum() <= 2


@pytest.mark.parametrize("which", ["x", "y", "dout", "p", "g", "m"])
def test_a_workspace_that_overlaps_the_calls_tensors_is_refused(which):
    """200 x 300 fp32 matrices (240000 bytes, more than a workgroup keeps in LDS), the workspace over the last 256 bytes of one of them."""
    L = md2amd._lib.lib(); size = 240000; at = {k: (i + 1) << 30 for i, k in enumerate(("x", "y", "dout", "p", "g", "m"))}; ws = (at[which] + size - 1) // 256 * 256
    st, co = (ctypes.c_int64 * 3)(60000, 300, 1), (ctypes.c_double * 3)(*COEF); V, I = ctypes.c_void_p, ctypes.c_int64
    if which in "pgm":
        r = L.md2_muon_raw((V * 1)(at["p"]), (V * 1)(at["g"]), (V * 1)(at["m"]), (I * 1)(200), (I * 1)(300), 1, 0.02, 0.95, 1, 0.0, 0, 1.0, 5, co, 1e-7, ws, 1 << 40, None)
    elif which == "dout":
        r = L.md2_newton_schulz_bwd(at["x"], at["dout"], at["y"], 1, 200, 300, st, st, 0, 5, co, 1e-7, ws, 1 << 40, None)
    else:
        r = L.md2_newton_schulz(at["x"], at["y"], 1, 200, 300, st, 0, 5, co, 1e-7, ws, 1 << 40, None)
    assert r == 2 and "workspace overlaps" in last_error()


def test_numbers_of_steps_that_no_int32_holds():
    m = md()
    for bad, passed in ((1 << 32 | 5, 17), (-(1 << 32) + 5, 0), (-3, 0), (0, 0), (17, 17), (5, 5), (16, 16), (5.0, 5)):
        assert m._ns_args(bad, COEF, 1e-7)[0] == passed
    for bad in (2.5, math.nan, math.inf):
        with pytest.raises((ValueError, OverflowError)):
            m._ns_args(bad, COEF, 1e-7)


@gpu
def test_muon_state_survives_a_shape_that_only_the_loss_takes():
    """An image too small for the network gives the model a loss-only handle for that call: the momentum passes through it, as ADAM's moments do."""
    m = md(); model, params, cache, x = make_model(); opt = m.Muon(eta=1e-3)
    m.train_step(model, x, None, cache, params, do_update=False); m.update(opt, model); st, adam, p = model.muon_state(), model._opt_and_bn_state(), model.params()
    H = W = 48; K, iK = md2amd.synthetic.depth10k_intrinsics(W, H); small = torch.from_numpy(md2amd.synthetic.synthetic_triplets(2, 1, H, W, seed=6)).cuda(); g = torch.Generator().manual_seed(5)
    cs = m.TrainCache(m.SSIM(), m.Backproject(W, H), m.Project(W, H), K, iK, 2, [1, 3], [0.125, 0.25, 0.5, 1.0]); model._ensure(small, m.Params(target_size=(W, H), batch_size=2, automasking=False), cs)
    disps = [(0.2 + 0.6 * torch.rand(2, 1, H >> k, W >> k, generator=g)).cuda() for k in (3, 2, 1, 0)]; r, t = [(0.01 * torch.randn(2, 2, 3, generator=g)).cuda() for _ in range(2)]
    assert np.isfinite(float(m.loss_fwd_bwd(model, small, disps, r, t)[0]))
    with pytest.raises(RuntimeError, match="loss-only"):
        m.update(opt, model)
    m.train_step(model, x, None, cache, params, do_update=False)
    assert np.array_equal(model.muon_state(), st) and np.array_equal(model.params(), p) and all(np.array_equal(a, b) for a, b in zip(model._opt_and_bn_state()[:4], adam[:4]))
    m.update(opt, model); assert not np.array_equal(model.muon_state(), st)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,pullback", [((5, 97, 211), 0), ((1, 512, 4608), 0), ((1, 512, 2304), 1), ((3, 385, 130), 1)])
def test_16_bit_results_are_roundings_of_results_as_accurate_as_fp32(shape, pullback, dtype):
    """Element by element: what is further from 64 bits than half a step of its type (fp16: of its subnormals, 2^-25) is so by no more than fp32's own error, whose root mean square the tests
    above bound by twice plain fp32's; the largest of 10^6 elements is held to eight times that.  Where two such results lie on both sides of a tie they differ by one step, and neither is the
    better one.  The same call gives the same bits."""
    m = md(); x = gradient_like(shape, sum(shape)).to(dtype).cuda(); d = torch.randn(shape, generator=torch.Generator().manual_seed(2), dtype=torch.float64).to(dtype).cuda()
    call = (lambda: m.newton_schulz_pullback(x, d)) if pullback else (lambda: m.newton_schulz(x))
    exact, plain = on_the_gpu(x, (lambda i, t: back_plain(x[i], d[i], 5, COEF, 1e-7, t)) if pullback else (lambda i, t: ns_plain(x[i].to(t))))
    y = call(); off = 8 * max(2 * rel(plain, exact), 4e-6 if pullback else 2e-6) * exact.square().mean().sqrt()
    assert ((y.double() - exact).abs() <= HALF[dtype] * (exact.abs() + off) + (2.0 ** -25 if dtype == torch.float16 else 0.0) + off).all()
    assert all(torch.equal(y, call()) for _ in range(5))
