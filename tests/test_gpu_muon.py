"""Newton-Schulz orthogonalisation and the Muon step against the formulas in 64 bits.

Tolerances.  To first order the result's error is the sum of what each rounding on the way adds, carried through the
rest of the polynomials, which depends on the spectrum.  So each test carries them through itself, in 64 bits: the chain
of products with the same groups of steps, once for each matrix that the operator stores, with that matrix M = U V
disturbed by random signs times the most that one of its entries can be off:
  r |M|          r half a step of how it is stored: 2^-12 ("half"), 2^-23 ("full"; both with f32 diagonals of Q, P,
                 which multiply X at 2^-23 in both)
  s |U| |V|      s = (4 + sqrt n) 2^-24: a float32 sum of n products whose roundings are independent, its epilogue, and
                 in "full" the product of the lo planes, at most 2^-24 of hi hi
and the norms and largest entries of the changes are added up, which is more than the root of the sum of their squares
that independent errors come to; the errors themselves are below those magnitudes, not at them.  What is stored
below f16's smallest step has that step instead; then the output is rounded to its type (half a step).
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

COEF = (3.4445, -4.7750, 2.0315)
V = 2.0 ** -24


def steps64(x, steps=5, eps=1e-7, coef=COEF, dtype=torch.float64):
    x = x.to(dtype)
    x = (x.double() / (x.double().square().sum().sqrt() + eps)).to(dtype)
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    for i in range(steps):
        a, b, c = coef[i] if isinstance(coef[0], tuple) else coef
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.t() if tall else x


def chain64(x, groups=(3, 2), eps=1e-7, coef=COEF, at=-1, r=0.0, signs=None):
    """The grouped steps; the result, and the number of matrices stored on the way, of which number ``at`` is off by
    signs times the magnitudes above."""
    x = x.double()
    x = x / (x.square().sum().sqrt() + eps)
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    stored = [0]

    def put(m, *factors, apart=False):
        stored[0] += 1
        if at != stored[0] - 1:
            return m
        off = r * (m - torch.diag(m.diagonal()) if apart else m).abs()
        if factors:
            u, v = factors
            off = off + (4 + u.shape[1] ** 0.5) * V * (u.abs() @ v.abs())
        sign = torch.randint(0, 2, m.shape, generator=signs, device=m.device) * 2 - 1
        return m + sign * off

    eye = torch.eye(x.shape[0], dtype=x.dtype, device=x.device)
    x, n = (put(x), x), 0  # as the products see it, and as the diagonals do
    for size in groups:
        g, p = put(x[0] @ x[0].t(), x[0], x[0].t()), None
        for i in range(size):
            a, b, c = coef[n] if isinstance(coef[0], tuple) else coef
            n += 1
            q = put(a * eye + b * g + c * (g @ g), c * g, g, apart=True)
            p = q if p is None else put(q @ p, q, p, apart=True)
            if i + 1 < size:
                t = put(q @ g, q, g)
                g = put(q @ t, q, t)
        d = p.diagonal()[:, None]
        y = (p - torch.diag(p.diagonal())) @ x[0] + d * x[1]
        x = (put(y, p, x[0]), y)
    x = x[0]
    return (x.t() if tall else x), stored[0]


def groups_of(steps, most):
    n = -(-steps // most)
    return [steps // n + (i < steps % n) for i in range(n)]


def tolerance(x, want, full, eps=1e-7, steps=5, coef=COEF, most=2):
    """(2-norm, largest) error allowed before the output is rounded, of one matrix."""
    S, L = min(x.shape), max(x.shape)
    groups = groups_of(steps, 3 if S <= 128 else 1 if L <= 1.25 * S else most)
    same, count = chain64(x, groups, eps, coef)
    assert (same - want).norm() <= 1e-9 * want.norm()  # the groups change nothing in exact arithmetic
    signs = torch.Generator(device=x.device).manual_seed(1)
    norm = top = 0.0
    for at in range(count):
        off = chain64(x, groups, eps, coef, at, 2.0 ** (-23 if full else -12), signs)[0] - want
        norm, top = norm + off.norm(), top + off.abs().max()
    # below f16's smallest step under the smallest scale in use, 2^-24 / 2^10, amplified by the last group (12)
    return norm + 1e-9 * want.numel() ** 0.5, 2 * top + 1e-8


def gradient(dev, E, M, N, rank, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 31 * E + 7 * M + N + rank)
    x = torch.randn(E, M, rank, generator=g) * torch.exp(torch.randn(E, 1, rank, generator=g))
    return (x @ torch.randn(E, rank, N, generator=g)).to(dtype).to(dev)


def held(got, x, full, u, eps=1e-7, steps=5, coef=COEF, which=None):
    for e in range(x.shape[0]) if which is None else which:
        want = steps64(x[e], steps, eps, coef)
        norm, top = tolerance(x[e], want, full, eps, steps, coef)
        off = got[e].double() - want
        assert torch.isfinite(off).all()
        assert off.norm() <= norm + u * want.norm(), (e, float(off.norm() / want.norm()), float(norm / want.norm()))
        assert (off.abs() <= top + u * want.abs()).all(), (e, float(off.abs().max()), float(top))


SIZES = [(1, 1, 1, 1), (2, 1, 5, 3), (3, 5, 1, 3), (4, 7, 3, 9), (2, 33, 31, 40), (3, 31, 65, 8), (2, 64, 200, 300),
         (2, 200, 64, 30), (8, 128, 512, 64), (3, 1001, 333, 500), (2, 300, 300, 600), (1, 257, 520, 1000),
         (1, 128, 128, 500), (2, 129, 1, 4), (1, 40, 2000, 16)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", SIZES)
def test_newton_schulz(dev, size, dtype):
    from mintext_amd.kernels import newton_schulz

    x = gradient(dev, *size, dtype)
    got = newton_schulz(x)
    assert got.dtype == dtype and got.shape == x.shape and got.is_contiguous()
    held(got, x, dtype == torch.float32, torch.finfo(dtype).eps / 2)


@pytest.mark.parametrize("precision", ["half", "full"])
@pytest.mark.parametrize("size", [(64, 264, 300, 500), (64, 300, 264, 100), (70, 512, 640, 700), (6, 1408, 1024, 2000)])
def test_many_and_large(dev, size, precision):
    """Sizes that run on the 256-row tiles, with tiles that hang over either side."""
    from mintext_amd.kernels import newton_schulz

    x = gradient(dev, *size, torch.bfloat16)
    E = size[0]
    got = newton_schulz(x.float(), precision=precision)
    held(got, x, precision == "full", V, which=sorted({0, 1, E // 2, E - 1}))
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("precision", ["half", "full"])
@pytest.mark.parametrize("size", [(80, 500, 548, 600), (80, 552, 504, 100), (80, 500, 704, 600), (80, 704, 504, 100)])
def test_large_tiles_hang_over(dev, size, precision):
    """Stacks with enough large tiles for the symmetric products too, whose last tile is not full."""
    from mintext_amd.kernels import newton_schulz

    x = gradient(dev, *size, torch.bfloat16)
    got = newton_schulz(x.float(), precision=precision)
    held(got, x, precision == "full", V, which=[0, 1, 40, 79])
    assert torch.isfinite(got).all()


def test_in_parts(dev):
    """A stack whose workspace would pass 4 GiB goes through in parts."""
    from mintext_amd import _lib as L
    from mintext_amd.kernels import newton_schulz

    E, M, N = 75, 2048, 2048
    assert L.query("mtx_newton_schulz_workspace_size", E, M, N, 1) < 4.1 * 2 ** 30
    assert E * (4 * M * N + 5 * M * N) * 2 > 4.1 * 2 ** 30
    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn(E, M, N, device=dev, generator=g).bfloat16()
    got = newton_schulz(x)
    held(got, x, False, 2.0 ** -8, which=[0, 37, 38, 74])


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7])
def test_steps_and_coefficients(dev, steps):
    from mintext_amd.kernels import newton_schulz

    x = gradient(dev, 2, 96, 160, 200, torch.float32)
    held(newton_schulz(x, steps), x, True, V, steps=steps)
    one = tuple((2.0 + 0.1 * i, -1.5, 0.5 - 0.02 * i) for i in range(steps))
    held(newton_schulz(x, steps, coefficients=one, eps=1e-3), x, True, V, 1e-3, steps, one)
    held(newton_schulz(x, steps, coefficients=(1.5, -0.5, 0.0), precision="half"), x, False, V, steps=steps,
         coef=(1.5, -0.5, 0.0))


def test_low_rank_and_decaying_spectra(dev):
    from mintext_amd.kernels import newton_schulz

    g = torch.Generator().manual_seed(11)
    u = torch.linalg.qr(torch.randn(160, 160, generator=g))[0]
    v = torch.linalg.qr(torch.randn(320, 160, generator=g))[0]
    x = torch.stack([(u * torch.logspace(0, -4, 160)) @ v.t(), (u * (1.0 / torch.arange(1, 161))) @ v.t(),
                     torch.randn(160, 2, generator=g) @ torch.randn(2, 320, generator=g)]).to(dev)
    for dtype in (torch.float32, torch.bfloat16):
        held(newton_schulz(x.to(dtype)), x.to(dtype), dtype == torch.float32, torch.finfo(dtype).eps / 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_zeros_nan_and_size_of_values(dev, dtype):
    from mintext_amd.kernels import newton_schulz

    x = gradient(dev, 6, 40, 72, 100, dtype)
    want = newton_schulz(x)
    y = x.clone()
    y[1] = 0
    y[3, 5, 7] = float("nan")
    y[4, 39, 71] = float("inf")
    got = newton_schulz(y)
    assert not got[1].any()
    assert torch.isnan(got[3]).all() and torch.isnan(got[4]).all()
    for e in (0, 2, 5):
        assert torch.equal(got[e], want[e])
    # powers of two move no rounding while eps is nothing beside the norm
    assert torch.equal(newton_schulz(x * 2.0 ** 60), newton_schulz(x * 2.0 ** 20))
    # a norm far below eps: nearly linear, a^5 x / eps
    small = x[:1] * 2.0 ** -40
    held(newton_schulz(small), small, dtype == torch.float32, torch.finfo(dtype).eps / 2)
    assert newton_schulz(x[:0]).shape == (0, 40, 72) and newton_schulz(x[:, :0]).shape == (6, 0, 72)


def test_strides(dev):
    from mintext_amd.kernels import newton_schulz

    x = gradient(dev, 4, 48, 72, 100, torch.bfloat16)
    want = newton_schulz(x)
    fused = torch.randn(4, 48, 200, device=dev).bfloat16()
    fused[:, :, 72:144] = x
    assert torch.equal(newton_schulz(fused[:, :, 72:144]), want)
    fused[:, :, 3:75] = x
    assert torch.equal(newton_schulz(fused[:, :, 3:75]), want)     # rows off a 16-byte boundary
    assert torch.equal(newton_schulz(x.permute(1, 0, 2).contiguous().permute(1, 0, 2)), want)
    assert torch.equal(newton_schulz(x.mT.contiguous().mT), want)  # copied
    assert torch.equal(newton_schulz(x[2:3].expand(3, 48, 72)), want[2:3].expand(3, 48, 72))
    assert torch.equal(newton_schulz(x.view(2, 2, 48, 72)), want.view(2, 2, 48, 72))
    assert torch.equal(newton_schulz(x[1]), want[1])


def step64(p, g, m, lr, beta, nesterov, wd, factor, full, eps=1e-7, steps=5):
    """(param, momentum) in 64 bits and their errors allowed, of one matrix."""
    u = torch.finfo(p.dtype).eps / 2
    m1 = beta * m.double() + (1 - beta) * g.double()
    x = (1 - beta) * g.double() + beta * m1 if nesterov else m1
    o = steps64(x, steps, eps)
    w = p.double() * (1 - lr * wd) - lr * factor * o
    norm, top = tolerance(x, o, full, eps, steps, most=3)
    # u and m are rounded to float32, beta and 1 - beta too: 4 half steps each, 2^-22, which is below twice what the
    # chain above allows the stored x in "full"
    size = beta * m.double().abs() + (1 - beta) * g.double().abs()
    tol_m = 4 * V * size
    tol = u * w.abs() + 4 * V * (p.double().abs() + lr * factor * o.abs())
    return w, m1, tol_m, (lr * factor * norm + tol.norm(), lr * factor * top + tol)


@pytest.mark.parametrize("types", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
                                   (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("size", [(1, 1, 1), (3, 40, 24), (2, 65, 130), (4, 128, 256), (2, 333, 200)])
def test_muon_update(dev, size, types):
    from mintext_amd.kernels import muon_update

    pt, gt = types
    E, M, N = size
    g = torch.Generator().manual_seed(sum(size))
    p = (torch.randn(*size, generator=g) * 0.02).to(pt).to(dev)
    m = torch.zeros(size, device=dev)
    lr, wd = 0.02, 0.1
    for step in range(3):
        nesterov, scale = step != 1, ("spectral", "rms", 0.3)[step]
        factor = max(1.0, N / M) ** 0.5 if step == 0 else 0.2 * max(M, N) ** 0.5 if step == 1 else 0.3
        grad = gradient(dev, E, M, N, 150, gt, seed=step)
        refs = [step64(p[e], grad[e], m[e], lr, 0.9, nesterov, wd, factor, pt == torch.float32) for e in range(E)]
        assert muon_update(p, grad, m, lr=lr, beta=0.9, nesterov=nesterov, weight_decay=wd, scale=scale) is p
        for e, (w, m1, tol_m, (norm, tol)) in enumerate(refs):
            assert ((m[e].double() - m1).abs() <= tol_m).all()
            off = p[e].double() - w
            assert off.norm() <= norm and (off.abs() <= tol).all(), (e, float(off.norm()), float(norm))


@pytest.mark.parametrize("pt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [(30, 200, 300), (30, 304, 200), (80, 500, 704), (80, 703, 504)])
def test_muon_update_of_many(dev, size, pt):
    """Stacks whose step runs on the middle (30) and on the large tiles (80); rows of whole 16-byte pieces, and not."""
    from mintext_amd.kernels import muon_update

    E, M, N = size
    g = torch.Generator().manual_seed(sum(size))
    p = (torch.randn(*size, generator=g) * 0.02).to(pt).to(dev)
    m = torch.randn(*size, generator=g).to(dev)
    grad = gradient(dev, E, M, N, 150, pt)
    which = [0, 1, E // 2, E - 1]
    refs = [step64(p[e], grad[e], m[e], 0.02, 0.9, True, 0.1, 0.3, pt == torch.float32) for e in which]
    muon_update(p, grad, m, lr=0.02, beta=0.9, weight_decay=0.1, scale=0.3)
    for e, (w, m1, tol_m, (norm, tol)) in zip(which, refs):
        assert ((m[e].double() - m1).abs() <= tol_m).all()
        off = p[e].double() - w
        assert off.norm() <= norm and (off.abs() <= tol).all(), (e, float(off.norm()), float(norm))
    assert torch.isfinite(p).all()


def test_muon_update_views(dev):
    """The halves of a fused stack step by themselves; the rest of it is not written."""
    from mintext_amd.kernels import muon_update

    g = torch.Generator(device=dev).manual_seed(5)
    fused = torch.randn(3, 64, 240, device=dev, generator=g).bfloat16()
    m = torch.randn(3, 64, 240, device=dev, generator=g)
    grad = torch.randn(3, 64, 240, device=dev, generator=g).bfloat16()
    for cols in (slice(0, 96), slice(96, 192), slice(5, 90)):
        w, mm = fused.clone(), m.clone()
        a, b = fused[:, :, cols].clone(), m[:, :, cols].clone()
        muon_update(w[:, :, cols], grad[:, :, cols], mm[:, :, cols], lr=0.1)
        muon_update(a, grad[:, :, cols].contiguous(), b, lr=0.1)
        assert torch.equal(w[:, :, cols], a) and torch.equal(mm[:, :, cols], b)
        w[:, :, cols], mm[:, :, cols] = fused[:, :, cols], m[:, :, cols]
        assert torch.equal(w, fused) and torch.equal(mm, m)
    # one matrix, and matrices that lie between each other's rows
    w = fused[0].clone()
    mix = fused.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    muon_update(w, grad[0], m[0].clone(), lr=0.1)
    muon_update(mix, grad, m.clone(), lr=0.1)
    assert torch.equal(mix[0], w)


def test_streams_and_graph(dev):
    """Another stream, the same bits again, and two captured steps with a learning rate on the device."""
    from mintext_amd.kernels import muon_update, newton_schulz

    x, y = (gradient(dev, 5, 130, 200, 100, torch.bfloat16, seed=s) for s in (0, 1))
    want, want_y = newton_schulz(x), newton_schulz(y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = newton_schulz(y)
    here = newton_schulz(x)  # at the same time
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(here, want) and torch.equal(other, want_y)

    p0, m0 = torch.randn(5, 130, 200, device=dev), torch.randn(5, 130, 200, device=dev)
    p, m, grad, lr = p0.clone(), m0.clone(), x.clone(), torch.tensor(0.02, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_update(p, grad, m, lr=lr, weight_decay=0.1)
    p.copy_(p0)
    m.copy_(m0)
    q, n = p0.clone(), m0.clone()
    for g, rate in ((x, 0.02), (y, 0.5), (x, 0.0), (y, 0.01)):
        grad.copy_(g)
        lr.fill_(rate)
        graph.replay()
        torch.cuda.synchronize()
        muon_update(q, g, n, lr=torch.tensor(rate, device=dev), weight_decay=0.1)
        assert torch.equal(p, q) and torch.equal(m, n)


def test_version_counters(dev):
    """Autograd sees that the weights changed under a saved forward."""
    from mintext_amd.kernels import linear, muon_update

    w = torch.randn(32, 32, device=dev).requires_grad_(True)
    y = linear(linear(torch.randn(8, 32, device=dev), w), w)
    muon_update(w, torch.randn(32, 32, device=dev), torch.zeros(32, 32, device=dev), lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_training_step_together(dev):
    """A dense layer and the experts of an MoE layer trained by their gradients: every weight moves as the formulas say."""
    from mintext_amd.kernels import grouped_matmul, linear, muon_update

    g = torch.Generator(device=dev).manual_seed(8)
    x = torch.randn(96, 64, device=dev, generator=g).bfloat16()
    w = (torch.randn(64, 128, device=dev, generator=g) * 0.1).bfloat16().requires_grad_(True)
    b = torch.zeros(128, device=dev, dtype=torch.bfloat16, requires_grad=True)
    experts = (torch.randn(4, 128, 64, device=dev, generator=g) * 0.1).bfloat16().requires_grad_(True)
    gs = torch.tensor([40, 0, 50, 6], dtype=torch.int32, device=dev)  # one expert without tokens
    y = grouped_matmul(linear(x, w, b, activation="silu"), experts, gs)
    gw, gb, ge = torch.autograd.grad(y, [w, b, experts], torch.randn(96, 64, device=dev, generator=g).bfloat16())
    for p, grad in ((w, gw), (experts, ge)):
        m = torch.zeros(p.shape, device=dev)
        before = p.detach().clone()
        muon_update(p, grad, m, lr=0.05, weight_decay=0.01)
        for e in range(1 if p.dim() == 2 else 4):
            pe, ge_, me = (t if p.dim() == 2 else t[e] for t in (before, grad, torch.zeros_like(m)))
            rows, cols = pe.shape
            want, _, _, (norm, tol) = step64(pe, ge_, me, 0.05, 0.95, True, 0.01, max(1.0, cols / rows) ** 0.5, False)
            off = (p.detach() if p.dim() == 2 else p.detach()[e]).double() - want
            assert off.norm() <= norm and (off.abs() <= tol).all()
