"""The dense product with its epilogue and its gradient against the formulas in 64 bits.

Tolerances, element by element.  u is the operands' half step (``finfo(t).eps / 2``), v that of float32.  A float32 sum
of n products is off by at most n v sum |a b|; the activations' slopes are at most 1.13 and their second
derivatives 0.8; a float32 activation or slope is allowed 16 half steps.  Hence
  dz_ = 1.13 (K + 2) v (|x| |w| + |b|)                                   the error of z
  y  : u |y| + dz_ + 16 v (|z| + |r|)
  ds : |dy| (0.8 (u |z| + dz_) + 16 v (1 + |z|)) + v |dz|                  dz before it is rounded, from the rounded z
  dx : u |dx| + (ds + u |dz|) |w|^T + N v |dz| |w|^T;  dw: alike;  db: u |db| + sum ds + M v sum |dz|
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

V = 2.0 ** -24
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]


def act64(z, act):
    f = torch.nn.functional
    return {None: lambda t: t, "relu": torch.relu, "silu": f.silu, "gelu": f.gelu,
            "gelu_tanh": lambda t: f.gelu(t, approximate="tanh")}[act](z)


def inputs(dev, T, K, N, dtype, bias, residual, seed=0):
    g = torch.Generator().manual_seed(seed + 7 * T + 3 * K + N)
    make = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(dtype).to(dev)
    return (make(T, K), make(K, N, std=max(K, 1) ** -0.5), make(N) if bias else None, make(T, N) if residual else None,
            make(T, N))


def reference(x, w, b, r, dy, act):
    leaves = [None if t is None else t.detach().double().requires_grad_(True) for t in (x, w, b, r)]
    z = leaves[0] @ leaves[1]
    z = z if b is None else z + leaves[2]
    z.retain_grad()
    y = act64(z, act)
    y = y if r is None else y + leaves[3]
    if dy is None:
        return z.detach(), y.detach(), None, None
    grads = torch.autograd.grad(y, [z] + [t for t in leaves if t is not None], dy.double())
    return z.detach(), y.detach(), grads[0], list(grads[1:])


def bounds(x, w, b, r, dy, act, z, y, dz, grads):
    u = torch.finfo(x.dtype).eps / 2
    ax, aw = x.detach().double().abs(), w.detach().double().abs()
    K, (M, N) = w.shape[0], y.shape
    size = ax @ aw + (0 if b is None else b.detach().double().abs())
    ez = 1.13 * (K + 2) * V * size
    ey = u * y.abs() + ez + 16 * V * (z.abs() + (0 if r is None else r.detach().double().abs()))
    if dy is None:
        return ey, None
    a = dy.double().abs()
    if act is None:
        es = torch.zeros_like(a)
    elif act == "relu":  # the slope is 0 or 1 except where the error of z reaches across 0
        es = torch.where(z.abs() <= ez, a, torch.zeros_like(a))
    else:
        es = a * (0.8 * (u * z.abs() + ez) + 16 * V * (1 + z.abs())) + V * dz.abs()
    er = es + (u * dz.abs() if act is not None else 0)
    out = [u * grads[0].abs() + er @ aw.t() + N * V * (dz.abs() @ aw.t()),
           u * grads[1].abs() + ax.t() @ er + M * V * (ax.t() @ dz.abs())]
    if b is not None:
        out.append(u * grads[2].abs() + es.sum(0) + M * V * dz.abs().sum(0))
    if r is not None:
        out.append(torch.zeros_like(a))
    return ey, out


def close(got, want, tol, what):
    assert got.shape == want.shape, what
    off = (got.double() - want).abs()
    bad = ~(off <= tol + 1e-40)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float((off / (tol + 1e-40)).max()):.2f} x"


def check(dev, T, K, N, dtype, act, bias, residual, train, seed=0):
    from mintext_amd.kernels import linear

    x, w, b, r, dy = inputs(dev, T, K, N, dtype, bias, residual, seed)
    if not train:
        dy = None
    z, y, dz, grads = reference(x, w, b, r, dy, act)
    ey, eg = bounds(x, w, b, r, dy, act, z, y, dz, grads)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r) if t is not None] if train else []
    out = linear(x, w, b, activation=act, residual=r)
    assert out.dtype == dtype
    close(out.detach(), y, ey, "y")
    if train:
        for name, got, want, tol in zip(("dx", "dw") + (("db",) if bias else ()) + (("dr",) if residual else ()),
                                        torch.autograd.grad(out, leaves, dy), grads, eg):
            assert got.dtype == dtype
            close(got, want, tol, name)


SIZES = [(1, 1, 1), (1, 8, 8), (3, 5, 7), (2, 40, 264), (17, 64, 24), (61, 1024, 320), (64, 33, 130), (129, 256, 264),
         (300, 520, 72), (257, 72, 520), (1000, 501, 250)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", SIZES)
def test_forward_and_gradients(dev, size, dtype):
    n = SIZES.index(size)
    check(dev, *size, dtype, ACTS[n % 5], n % 2 == 0, n % 3 != 0, True)
    check(dev, *size, dtype, ACTS[(n + 2) % 5], n % 2 == 1, n % 3 == 0, False, seed=1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", ACTS)
def test_activations(dev, act, dtype):
    check(dev, 77, 136, 200, dtype, act, True, True, True)
    check(dev, 9, 136, 200, dtype, act, False, False, True)


@pytest.mark.parametrize("size", [(1, 4096, 1024), (1, 14336, 256), (16, 2048, 1408), (40, 7168, 768)])
def test_few_rows(dev, size):
    check(dev, *size, torch.bfloat16, "silu", True, True, False)
    check(dev, *size, torch.bfloat16, None, False, False, False)


@pytest.mark.parametrize("size", [(1531, 1536, 704), (2048, 2048, 768), (1025, 4096, 1288), (4099, 512, 2056),
                                  (8192, 128, 256), (130, 7168, 2048), (4099, 520, 2056), (4099, 72, 4104),
                                  (300, 4104, 4104)])
def test_large(dev, size):
    n = size[0] % 5
    check(dev, *size, torch.bfloat16, ACTS[n], True, n % 2 == 0, True)


@pytest.mark.parametrize("size", [(3330, 136, 2056), (3330, 128, 2056), (3330, 2056, 136), (3330, 2056, 128),
                                  (150, 3336, 2056), (96, 3336, 2056), (4099, 2056, 72), (5000, 264, 2056)])
def test_each_product_in_each_tile(dev, size):
    """The forward product and both gradients in middle and in large tiles that hang over, with whole and cut stages."""
    check(dev, *size, torch.bfloat16, "silu", True, False, True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_empty(dev, dtype):
    from mintext_amd.kernels import linear

    w, b = torch.randn(8, 16, device=dev, dtype=dtype), torch.randn(16, device=dev, dtype=dtype)
    x = torch.randn(0, 8, device=dev, dtype=dtype, requires_grad=True)
    w.requires_grad_(True)
    y = linear(x, w, b, activation="silu")
    assert y.shape == (0, 16)
    dx, dw = torch.autograd.grad(y, [x, w], torch.zeros_like(y))
    assert dx.shape == (0, 8) and not dw.any()
    # no reduction: the bias alone
    y = linear(torch.randn(3, 0, device=dev, dtype=dtype), torch.randn(0, 16, device=dev, dtype=dtype), b)
    assert torch.equal(y, b.expand(3, 16))


@pytest.mark.parametrize("act", ["relu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("size", [(40, 64, 72), (300, 64, 256), (40, 33, 70)])
def test_infinities_and_nan(dev, act, size):
    """They reach the outputs that they reach in the formula, and no other."""
    from mintext_amd.kernels import linear

    T, K, N = size
    x, w, b, r, _ = inputs(dev, T, K, N, torch.bfloat16, True, True)
    x[3, 5], x[T - 1, K - 1], w[2, 4], b[7], r[1, 9] = float("inf"), float("nan"), float("-inf"), float("inf"), float("nan")
    _, y, _, _ = reference(x, w, b, r, None, act)
    out = linear(x, w, b, activation=act, residual=r).double()
    assert torch.equal(torch.isnan(out), torch.isnan(y)) and torch.equal(torch.isinf(out), torch.isinf(y))
    fine = torch.isfinite(y)
    assert (out[fine] - y[fine]).abs().max() <= 2.0 ** -6 * y[fine].abs().max()


def test_shapes_strides_and_alignment(dev):
    """Leading dimensions, transposed and sliced operands, an expanded residual, tensors off a 16-byte boundary."""
    from mintext_amd.kernels import linear

    g = torch.Generator(device=dev).manual_seed(3)
    t = torch.bfloat16
    x = torch.randn(64, 4, 6, device=dev, generator=g).to(t).permute(2, 1, 0)  # [6, 4, 64]
    w = torch.randn(80, 64, device=dev, generator=g).to(t).t()
    b = torch.randn(160, device=dev, generator=g).to(t)[::2]
    r = torch.randn(80, device=dev, generator=g).to(t).expand(6, 4, 80)
    want = linear(x.contiguous(), w.contiguous(), b.contiguous(), activation="silu", residual=r.contiguous())
    assert torch.equal(linear(x, w, b, activation="silu", residual=r), want)
    flat = torch.empty(1 + 24 * 64, device=dev, dtype=t)
    off = flat[1:].view(6, 4, 64).copy_(x)
    z, y, _, _ = reference(off.reshape(24, 64), w, b, r.reshape(24, 80), None, "silu")
    ey, _ = bounds(off.reshape(24, 64), w, b, r.reshape(24, 80), None, "silu", z, y, None, None)
    close(linear(off, w, b, activation="silu", residual=r).reshape(24, 80), y, ey, "off a 16-byte boundary")
    # a gradient that is an expanded scalar, and one that is transposed
    x2, w2 = (v.detach().contiguous().requires_grad_(True) for v in (x.reshape(24, 64), w))
    gx, gw = torch.autograd.grad(linear(x2, w2, activation="gelu").sum(), [x2, w2])
    hx, hw = torch.autograd.grad(linear(x2, w2, activation="gelu"), [x2, w2], torch.ones(80, 24, device=dev, dtype=t).t())
    assert torch.equal(gx, hx) and torch.equal(gw, hw)


def test_broadcast_inputs_gradients(dev):
    """A residual that is broadcast and a weight that is used twice get the sums of their gradients."""
    from mintext_amd.kernels import linear

    g = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn(50, 64, device=dev, generator=g)
    w = torch.randn(64, 64, device=dev, generator=g).mul_(0.1).requires_grad_(True)
    r = torch.randn(64, device=dev, generator=g).requires_grad_(True)
    y = linear(linear(x, w, activation="silu"), w, residual=r.expand(50, 64))
    gw, gr = torch.autograd.grad(y.sum(), [w, r])
    w64, r64 = w.detach().double().requires_grad_(True), r.detach().double().requires_grad_(True)
    y64 = torch.nn.functional.silu(x.double() @ w64) @ w64 + r64
    hw, hr = torch.autograd.grad(y64.sum(), [w64, r64])
    # two products of 64 terms each behind one another: 4 * 66 half steps of the terms' sizes (below 40)
    assert (gw.double() - hw).abs().max() <= 4 * 66 * V * hw.abs().max() * 4
    assert torch.equal(gr.double(), hr)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gradient_against_differences(dev, act):
    from mintext_amd.kernels import linear

    T, K, N, h = 20, 48, 72, 2.0 ** -5
    x, w, b, r, dy = inputs(dev, T, K, N, torch.float32, True, True)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
    grads = torch.autograd.grad(linear(x, w, b, activation=act, residual=r), leaves, dy)
    g = torch.Generator().manual_seed(9)
    for n, leaf in enumerate(leaves):
        d = torch.randn(*leaf.shape, generator=g).to(dev) * (0.1 if n == 1 else 1.0)
        at = lambda s: [t.detach() + (s * h * d if i == n else 0) for i, t in enumerate(leaves)]
        f = lambda s: (linear(*at(s)[:3], activation=act, residual=at(s)[3]).double() * dy.double()).sum()
        slope = (f(1) - f(-1)) / (2 * h)
        want = (grads[n].double() * d.double()).sum()
        # third derivatives stay below 2: h^2 / 6 * 2 |dy| |dz/dt|^3; float32 outputs of size below 64, off by K + 18
        # half steps each, divided by h
        move = d.double() @ w.double() if n == 0 else x.double() @ d.double() if n == 1 else d.double().expand(T, N)
        tol = h * h / 3 * (dy.double().abs() * move.detach().abs() ** 3).sum()
        tol = tol + dy.double().abs().sum() * (K + 18) * V * 64 / h
        assert (slope - want).abs() <= tol, (n, float(slope), float(want), float(tol))


def test_only_what_is_asked_for(dev):
    from mintext_amd.kernels import linear

    x, w, b, r, dy = inputs(dev, 30, 64, 64, torch.bfloat16, True, True)
    for leaf in (x, w, b, r):
        leaf.requires_grad_(True)
        y = linear(x, w, b, activation="gelu", residual=r)
        (only,) = torch.autograd.grad(y, [leaf], dy)
        leaf.requires_grad_(False)
        full = [t.detach().clone().requires_grad_(True) for t in (x, w, b, r)]
        every = torch.autograd.grad(linear(*full[:3], activation="gelu", residual=full[3]), full, dy)
        assert torch.equal(only, every[[id(t) for t in (x, w, b, r)].index(id(leaf))])
    y = linear(x.requires_grad_(True), w, activation="silu")
    (gx,) = torch.autograd.grad(y.sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.sum(), [x])


@pytest.mark.parametrize("size", [(1, 512, 256), (37, 2048, 768), (700, 512, 520), (50, 33, 70)])
def test_streams_and_graph(dev, size):
    """Another stream, repeated calls bit for bit, and a captured call replayed between eager ones."""
    from mintext_amd.kernels import linear

    x, w, b, r, _ = inputs(dev, *size, torch.bfloat16, True, True)
    x2 = torch.flip(x, [1]).contiguous()
    call = lambda t: linear(t, w, b, activation="silu", residual=r)
    want, want2 = call(x), call(x2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(call(x), want)
    torch.cuda.current_stream().wait_stream(side)
    held = x.clone()
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(held)
    with torch.cuda.graph(graph2, pool=graph.pool()):
        out2 = call(held)
    for t, y in ((x, want), (x2, want2), (x, want), (x2, want2)):
        held.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, y) and torch.equal(call(t), y)
        graph2.replay()
        torch.cuda.synchronize()
        assert torch.equal(out2, y)


def test_with_the_grouped_product(dev):
    """One group of the grouped product is the same product."""
    from mintext_amd.kernels import grouped_matmul, linear

    x, w, _, _, _ = inputs(dev, 200, 256, 512, torch.bfloat16, False, False)
    gs = torch.tensor([200], dtype=torch.int32, device=dev)
    a, b = linear(x, w).double(), grouped_matmul(x, w[None], gs).double()
    # each rounds its own f32 sum once
    assert ((a - b).abs() <= 2 * 2.0 ** -8 * b.abs() + 2 * 258 * V * (x.double().abs() @ w.double().abs())).all()
