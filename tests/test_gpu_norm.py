"""The norms and their gradients against the formulas in 64 bits.

Tolerances, element by element.  u is the half step of a result's type (``finfo(t).eps / 2``), v that of float32.  A sum over a
row is 16 additions in a lane, 6 between lanes and at most 16 between waves: off by at most 40 v of its terms' sizes.
  em = 42 v mean|h|                                the mean; then of rstd, relative:
  er = 30 v + em^2 / (2 (var + eps))               (half of 44 v of the squares, division and root 8 v; the mean's error adds em^2)
  en = rstd (em + |d| (er + 4 v))                  n = d rstd
  y  : u |y| + |w| en + 2 v (|n w| + |b|)
  dx : rstd (3 v |u| + 44 v mean|u| + |n| ec + |c| en + 4 v |n c|) + |dx - dh| (er + 4 v) + 2 v |dh| + u |dx|,
       u = dy w, c = mean(u n), ec = 44 v mean|u n| + mean(|u| en)
  dw : u |dw| + sum_t |dy| en + (T + 2) v sum_t |dy n|;  db: u |db| + T v sum_t |dy|
The sum h is rounded once from float32 and has to be equal.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

V = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32


def inputs(dev, T, D, dtype, wtype, bias, residual, seed=0):
    g = torch.Generator().manual_seed(seed + 7 * T + D)
    make = lambda *s, std=1.0, mean=0.0, t=dtype: (torch.randn(*s, generator=g) * std + mean).to(t).to(dev)
    x = make(T, D, mean=0.5)
    if D > 2:
        x[:, 1] *= 30  # a feature that is far off
    return (x, make(T, D, std=2.0) if residual else None, make(D, std=0.3, mean=1.0, t=wtype),
            make(D, t=wtype) if bias else None, make(T, D), make(T, D) if residual else None)


def reference(x, r, w, b, dy, dh, rms, eps):
    """h, and in 64 bits y, dx, dw, db with their tolerances."""
    u = torch.finfo(x.dtype).eps / 2
    uw = torch.finfo(w.dtype).eps / 2
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    H, W, DY = h.double(), w.double(), dy.double()
    mean = torch.zeros_like(H[:, :1]) if rms else H.mean(1, keepdim=True)
    d = H - mean
    var = (d * d).mean(1, keepdim=True)
    rstd = (var + eps) ** -0.5
    n = d * rstd
    em = 0 * var if rms else 42 * V * H.abs().mean(1, keepdim=True)
    er = 30 * V + em * em / (2 * (var + eps))
    en = rstd * (em + d.abs() * (er + 4 * V))
    y = n * W if b is None else n * W + b.double()
    ty = u * y.abs() + W.abs() * en + 2 * V * ((n * W).abs() + (0 if b is None else b.double().abs()))
    U = DY * W
    c = (U * n).mean(1, keepdim=True)
    m = torch.zeros_like(c) if rms else U.mean(1, keepdim=True)
    core = rstd * (U - m - n * c)
    dx = core if dh is None else core + dh.double()
    ec = 44 * V * (U * n).abs().mean(1, keepdim=True) + (U.abs() * en).mean(1, keepdim=True)
    tx = rstd * (3 * V * U.abs() + 44 * V * U.abs().mean(1, keepdim=True) + n.abs() * ec + c.abs() * en + 4 * V * (n * c).abs())
    tx = tx + core.abs() * (er + 4 * V) + u * dx.abs() + (0 if dh is None else 2 * V * dh.double().abs())
    dw, db = (DY * n).sum(0), DY.sum(0)
    tw = uw * dw.abs() + (DY.abs() * en).sum(0) + (len(x) + 2) * V * (DY * n).abs().sum(0)
    tb = uw * db.abs() + len(x) * V * DY.abs().sum(0)
    return h, (y, ty), (dx, tx), (dw, tw), (db, tb)


def close(got, want, what):
    want, tol = want
    assert got.shape == want.shape, what
    off = (got.double() - want).abs()
    bad = ~(off <= tol + 1e-40)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float((off / (tol + 1e-40)).max()):.2f} x"


def call(x, r, w, b, rms, eps):
    from mintext_amd.kernels import layer_norm, rms_norm

    return rms_norm(x, w, eps=eps, residual=r) if rms else layer_norm(x, w, b, eps=eps, residual=r)


def check(dev, T, D, dtype, wtype, rms, bias, residual, seed=0, eps=1e-5):
    x, r, w, b, dy, dh = inputs(dev, T, D, dtype, wtype, bias and not rms, residual, seed)
    h, y, dx, dw, db = reference(x, r, w, b, dy, dh, rms, eps)
    out = call(x, r, w, b, rms, eps)
    leaves = [t.requires_grad_(True) for t in (x, r, w, b) if t is not None]
    train = call(x, r, w, b, rms, eps)
    out, train = ([out], [train]) if r is None else (out, train)
    assert all(torch.equal(a, t.detach()) for a, t in zip(out, train))
    assert out[0].dtype == dtype
    close(out[0], y, "y")
    if r is not None:
        assert torch.equal(out[1], h)
    grads = torch.autograd.grad(list(train), leaves, [dy] + ([dh] if r is not None else []))
    names = ["dx"] + (["dr"] if r is not None else []) + ["dw"] + (["db"] if b is not None else [])
    wants = [dx] + ([dx] if r is not None else []) + [dw] + ([db] if b is not None else [])
    for name, got, want, leaf in zip(names, grads, wants, leaves):
        assert got.dtype == leaf.dtype, name
        close(got, want, name)


# each number of waves a row, whole, hanging over and odd; one row, a row more or less than a workgroup takes, many
SIZES = [(1, 1), (3, 7), (1, 8), (17, 24), (5, 501), (33, 1000), (64, 1024), (300, 1032), (257, 2048), (9, 2047), (130, 4096),
         (1030, 3001), (1025, 4104), (2, 7168), (515, 8192), (259, 8191), (40, 8200), (300, 16384), (33, 16383)]


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("size", SIZES)
def test_forward_and_gradients(dev, size, dtype, rms):
    n = SIZES.index(size)
    check(dev, *size, dtype, dtype, rms, n % 2 == 0, n % 3 == 0)
    check(dev, *size, dtype, F32, rms, n % 2 == 1, n % 3 != 0, seed=1)


@pytest.mark.parametrize("rms", [False, True])
def test_many_rows(dev, rms):
    check(dev, 20000, 136, BF, BF, rms, True, True)
    check(dev, 9001, 4096, BF, F32, rms, True, True)


def test_more_rows_than_a_grid_holds(dev):
    """D = 1: rms_norm(x) = x / sqrt(x^2 + eps) w, to be within a few roundings of float32 and one of bfloat16."""
    from mintext_amd.kernels import rms_norm

    T = 2 ** 28 + 2 ** 20 + 3
    x = torch.empty(T, 1, device=dev, dtype=torch.bfloat16)
    x.view(-1)[::2], x.view(-1)[1::2] = 0.75, -1.5
    x[0], x[2 ** 28 - 1], x[2 ** 28], x[T - 1] = 3.0, 0.0, 0.01, -7.0
    w = torch.full((1,), 1.25, device=dev, dtype=torch.bfloat16)
    y = rms_norm(x, w, eps=1e-3)
    for at in (slice(0, 4), slice(2 ** 28 - 4, 2 ** 28 + 4), slice(T - 4, T)):
        X = x[at].double()
        want = X / (X * X + 1e-3).sqrt() * 1.25
        assert ((y[at].double() - want).abs() <= (2.0 ** -8 + 8 * 2.0 ** -24) * want.abs()).all()
    # 1.25 and -1.25 in bfloat16, of 3 and -7 too
    assert int((y == 1.25).sum() + (y == -1.25).sum()) == T - 2


@pytest.mark.parametrize("eps", [0.0, 1e-12, 1.0])
def test_eps_and_constant_rows(dev, eps):
    check(dev, 10, 64, F32, F32, False, True, False, eps=eps)
    x = torch.full((4, 64), 3.0, device=dev)
    w, b = torch.ones(64, device=dev), torch.full((64,), 0.25, device=dev)
    y = call(x, None, w, b, False, eps)
    assert torch.equal(y, b.expand(4, 64)) if eps > 0 else torch.isnan(y).all()


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("D", [64, 65])
def test_infinities_and_nan_stay_in_their_row(dev, rms, D):
    x, _, w, b, dy, _ = inputs(dev, 20, D, BF, BF, not rms, False)
    clean = call(x, None, w, b, rms, 1e-5)
    x2 = x.clone()
    x2[3, 5], x2[7, 2], x2[19, D - 1] = float("inf"), float("nan"), float("-inf")
    out = call(x2, None, w, b, rms, 1e-5)
    bad = torch.tensor([3, 7, 19], device=dev)
    keep = torch.ones(20, dtype=torch.bool, device=dev)
    keep[bad] = False
    assert torch.equal(out[keep], clean[keep]) and torch.isnan(out[bad]).any(1).all()


def test_empty(dev):
    from mintext_amd.kernels import layer_norm

    x = torch.empty(0, 40, device=dev, requires_grad=True)
    w, b = torch.ones(40, device=dev, requires_grad=True), torch.ones(40, device=dev, requires_grad=True)
    y, h = layer_norm(x, w, b, residual=torch.empty(0, 40, device=dev))
    dx, dw, db = torch.autograd.grad([y, h], [x, w, b], [torch.empty_like(y), torch.empty_like(h)])
    assert y.shape == h.shape == dx.shape == (0, 40) and not dw.any() and not db.any()


def test_shapes_strides_and_alignment(dev):
    from mintext_amd.kernels import layer_norm

    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn(64, 4, 6, device=dev, generator=g).to(BF).permute(2, 1, 0)
    w = torch.randn(128, device=dev, generator=g).to(BF)[::2]
    b = torch.randn(1, device=dev, generator=g).to(BF).expand(64)
    want = layer_norm(x.contiguous(), w.contiguous(), b.contiguous())
    assert torch.equal(layer_norm(x, w, b), want)
    flat = torch.empty(1 + 24 * 64, device=dev, dtype=BF)
    off = flat[1:].view(6, 4, 64).copy_(x)
    _, y, _, _, _ = reference(off.reshape(24, 64), None, w, b, off.reshape(24, 64), None, False, 1e-5)
    close(layer_norm(off, w, b).reshape(24, 64), y, "off a 16-byte boundary")
    # gradients that are an expanded scalar and a transposed tensor
    x2 = x.contiguous().requires_grad_(True)
    (gx,) = torch.autograd.grad(layer_norm(x2, w, b).sum(), [x2])
    ones = torch.ones(64, 4, 6, device=dev, dtype=BF).permute(2, 1, 0)
    (hx,) = torch.autograd.grad(layer_norm(x2, w, b), [x2], ones)
    assert torch.equal(gx, hx)


def test_only_what_is_asked_for(dev):
    x, r, w, b, dy, dh = inputs(dev, 30, 72, BF, BF, True, True)
    every = [t.detach().clone().requires_grad_(True) for t in (x, r, w, b)]
    full = torch.autograd.grad(list(call(every[0], every[1], every[2], every[3], False, 1e-5)), every, [dy, dh])
    for n, leaf in enumerate((x, r, w, b)):
        leaf.requires_grad_(True)
        (only,) = torch.autograd.grad(list(call(x, r, w, b, False, 1e-5)), [leaf], [dy, dh])
        leaf.requires_grad_(False)
        assert torch.equal(only, full[n])
    # one of the two results alone
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, r, w, b)]
    y, h = call(*leaves, False, 1e-5)
    gx, gr, gw, gb = torch.autograd.grad(h, leaves, dh, retain_graph=True, allow_unused=True)
    assert torch.equal(gx, dh) and torch.equal(gr, dh) and gw is None and gb is None
    got = torch.autograd.grad(y, leaves, dy)
    zero = torch.autograd.grad(list(call(*leaves, False, 1e-5)), leaves, [dy, torch.zeros_like(dh)])
    assert all(torch.equal(a, c) for a, c in zip(got, zero))
    (gx,) = torch.autograd.grad(call(leaves[0], None, leaves[2], leaves[3], False, 1e-5).sum(), [leaves[0]], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.sum(), [leaves[0]])


def test_a_tensor_beside_itself(dev):
    """x as its own residual gets both gradients; a weight used twice the sum of its two."""
    x, _, w, b, dy, dh = inputs(dev, 20, 72, F32, F32, True, True)
    other = x.detach().clone().requires_grad_(True)
    x.requires_grad_(True), w.requires_grad_(True)
    (gx,) = torch.autograd.grad(list(call(x, x, w, b, False, 1e-5)), [x], [dy, dh])
    parts = torch.autograd.grad(list(call(x, other, w, b, False, 1e-5)), [x, other], [dy, dh])
    assert torch.equal(gx, parts[0] + parts[1])
    y1, y2 = call(x, None, w, b, False, 1e-5), call(dh, None, w, b, False, 1e-5)
    (gw,) = torch.autograd.grad([y1, y2], [w], [dy, dy], retain_graph=True)
    (g1,) = torch.autograd.grad(y1, [w], dy)
    (g2,) = torch.autograd.grad(y2, [w], dy)
    assert torch.equal(gw, g1 + g2)


@pytest.mark.parametrize("rms", [False, True])
def test_gradient_against_differences(dev, rms):
    """The slope along a random direction, of the formula in 64 bits: a step of 1e-5 leaves 1e-10 of third derivatives (values
    below 1e3) and 1e-16 / 1e-5 of rounding, of sums of size below 1e4."""
    T, D, step, eps = 6, 40, 1e-5, 1e-5
    x, r, w, b, dy, dh = inputs(dev, T, D, F32, F32, not rms, True)
    _, _, tx, tw, tb = reference(x, r, w, b, dy, dh, rms, eps)
    leaves = [t.requires_grad_(True) for t in (x, r, w, b) if t is not None]
    grads = torch.autograd.grad(list(call(x, r, w, b, rms, eps)), leaves, [dy, dh])
    g = torch.Generator().manual_seed(9)
    for n, (leaf, tol) in enumerate(zip(leaves, (tx, tx, tw, tb))):
        move = torch.randn(*leaf.shape, generator=g).to(dev).double()

        def f(s):
            at = [t.detach().double() + (s * step * move if i == n else 0) for i, t in enumerate(leaves)]
            h = at[0] + at[1]
            d = h if rms else h - h.mean(1, keepdim=True)
            y = d / ((d * d).mean(1, keepdim=True) + eps).sqrt() * at[2] + (0 if rms else at[3])
            return (y * dy.double()).sum() + (h * dh.double()).sum()

        slope, want = (f(1) - f(-1)) / (2 * step), (grads[n].double() * move).sum()
        # h of the kernel is rounded to float32: half a step of at most 256, which the norm's slopes (below 10) carry on
        allowed = (tol[1] * move.abs()).sum() + 1e-6 * (1 + (tol[0] * move).abs().sum()) + 10 * V * 256 * dy.double().abs().sum()
        assert (slope - want).abs() <= allowed, (n, float(slope), float(want), float(allowed))


@pytest.mark.parametrize("size", [(1, 512), (700, 2048), (50, 33)])
def test_streams_and_graph(dev, size):
    """Another stream, repeated calls bit for bit, and a captured step replayed between eager ones."""
    x, r, w, b, dy, dh = inputs(dev, *size, BF, BF, True, True)
    x2 = torch.flip(x, [1]).contiguous()

    def step(t):
        leaves = [v.detach().requires_grad_(True) for v in (t, r, w, b)]  # leaves of its own: no graph outlives a call
        out = call(*leaves, False, 1e-5)
        return [o.detach() for o in out] + list(torch.autograd.grad(list(out), leaves, [dy, dh]))

    same = lambda a, c: all(torch.equal(i, j) for i, j in zip(a, c))
    want, want2 = step(x), step(x2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert same(step(x), want)
    torch.cuda.current_stream().wait_stream(side)
    held = x.clone()
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held)
    with torch.cuda.graph(graph2, pool=graph.pool()):
        out2 = step(held)
    for t, y in ((x, want), (x2, want2), (x, want), (x2, want2)):
        held.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, y) and same(step(t), y)
        graph2.replay()
        torch.cuda.synchronize()
        assert same(out2, y)


def test_jit_trace_computes(dev):
    from mintext_amd.kernels import layer_norm

    w, b = torch.randn(64, device=dev), torch.randn(64, device=dev)
    f = lambda x: layer_norm(x, w, b)
    a, c = torch.randn(10, 64, device=dev), torch.randn(10, 64, device=dev)
    assert torch.equal(torch.jit.trace(f, (a,), check_trace=False)(c), f(c))
