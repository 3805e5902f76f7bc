"""Float32 results of ``newton_schulz`` are rounded once: products and sums are in float64.

Tolerance: half a step of the result, and 1e-9 of its norm for everything in 64 bits (a sum of up to 2000 terms is off by
2^-53 sqrt(2000) of them, and the five steps carry that up by 3.4445^5 = 485 at most: 3e-12; the coefficients are held
to 2^-49, eps to 2^-25 of itself, which is nothing beside a norm above 1e-2).
"""
from __future__ import annotations

import pytest
import torch
from test_gpu_muon import steps64
from test_muon_groups import STEEP, gradient

pytestmark = pytest.mark.gpu


def check(got, x, steps=5, coef=(3.4445, -4.7750, 2.0315), eps=1e-7):
    for e in {0, len(x) // 2, len(x) - 1}:
        want = steps64(x[e], steps, eps, coef)
        off = (got[e].double() - want).abs()
        assert (off <= torch.finfo(got.dtype).eps / 2 * want.abs() + 1e-9 * want.norm()).all(), (e, float(off.max()))


# few and many matrices: tiles of 32 x 32 and of 64 x 64, whole and hanging over
SIZES = [(1, 1, 1), (3, 1, 5), (3, 5, 1), (2, 33, 31), (2, 31, 65), (8, 128, 512), (2, 300, 300), (3, 333, 150), (1, 40, 2000),
         (1, 2000, 33), (80, 200, 321), (80, 321, 200), (600, 64, 64), (40, 500, 200)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", SIZES)
def test_sizes(dev, size, dtype):
    from mintext_amd.kernels import newton_schulz

    E, M, N = size
    x = torch.stack([gradient(M, N, r) for r in (1, 3, max(M, N))])[torch.arange(E) % 3].to(dtype).to(dev)
    got = newton_schulz(x, precision="double")
    check(got, x)
    if dtype == torch.float32:
        assert torch.equal(newton_schulz(x), got)


@pytest.mark.parametrize("size", [(768, 768, 32), (700, 768, 32), (512, 512, 64), (128, 512, 1)])
def test_low_ranks(dev, size):
    """Two f16 planes and float32 sums end 2e-5 to 1e-4 off here."""
    from mintext_amd.kernels import newton_schulz

    x = gradient(*size)[None].to(dev)
    check(newton_schulz(x), x)


@pytest.mark.parametrize("coef", [(1.5, -0.5, 0.0), (1.25, 0.0, -0.25), (1.0, -1e-3, 1e-6), STEEP],
                         ids=["cubic", "even", "faint", "steep"])
@pytest.mark.parametrize("steps", [1, 2, 5])
def test_coefficients_and_steps(dev, steps, coef):
    from mintext_amd.kernels import newton_schulz

    coef = coef[:steps] if isinstance(coef[0], tuple) else coef
    for size in ((90, 200, 100), (200, 90, 100)):
        x = gradient(*size)[None].to(dev)
        check(newton_schulz(x, steps, coefficients=coef, eps=2.0 ** -10), x, steps, coef, 2.0 ** -10)


def test_zeros_nan_infinities_and_strides(dev):
    from mintext_amd.kernels import newton_schulz

    x = torch.stack([gradient(40, 72, 100)] * 5).to(dev)
    want = newton_schulz(x)
    y = torch.zeros(5, 40, 80, device=dev)[..., 3:75].copy_(x)
    y[1], y[2, 3, 4], y[3, 5, 6] = 0, float("nan"), float("-inf")
    got = newton_schulz(y)
    assert torch.equal(got[0], want[0]) and torch.equal(got[4], want[4]) and not got[1].any()
    assert torch.isnan(got[2]).all() and torch.isnan(got[3]).all()
    assert torch.equal(newton_schulz(x.mT).mT, newton_schulz(x.mT.contiguous()).mT)
    tiny = x[:1] * 2.0 ** -60  # nearly linear: eps is the norm, and held in float32
    assert torch.isfinite(newton_schulz(tiny)).all()


def test_in_parts(dev):
    """A stack whose workspace would pass 4 GiB."""
    from mintext_amd import _lib as L
    from mintext_amd.kernels import newton_schulz

    E, M, N = 600, 300, 1400
    assert L.query("mtx_newton_schulz_workspace_size", E, M, N, L.MTX_NS_F64) < 4.1 * 2 ** 30
    assert E * 16 * (M * N + M * M) > 4.1 * 2 ** 30
    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn(E, M, N, device=dev, generator=g)
    got = newton_schulz(x)
    for e in (0, 299, 300, 599):
        check(got[e:e + 1], x[e:e + 1])


@pytest.mark.parametrize("types", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
                                   (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("size", [(1, 1, 1), (3, 40, 24), (2, 65, 130), (30, 200, 304)])
def test_muon_update(dev, size, types):
    from mintext_amd.kernels import muon_update

    pt, gt = types
    E, M, N = size
    g = torch.Generator().manual_seed(sum(size))
    p = (torch.randn(*size, generator=g) * 0.02).to(pt).to(dev)
    m = torch.randn(*size, generator=g).to(dev)
    grad = torch.randn(*size, generator=g).to(gt).to(dev)
    lr, wd, beta = 0.0625, 0.125, 0.75  # held in float32 as they are
    m1 = beta * m.double() + (1 - beta) * grad.double()
    u = (1 - beta) * grad.double() + beta * m1
    want = [p[e].double() * (1 - lr * wd) - lr * 0.5 * steps64(u[e]) for e in range(E)]
    muon_update(p, grad, m, lr=torch.tensor(lr, device=dev), beta=beta, weight_decay=wd, scale=0.5, precision="double")
    # m and u are rounded to float32, two half steps each of their terms; that moves the orthogonalised matrix by at most
    # 485 (the steps' largest slope) times as much in the 2-norm
    for e in range(E):
        off = (p[e].double() - want[e]).norm()
        assert off <= torch.finfo(pt).eps / 2 * want[e].norm() + lr * 0.5 * 485 * 4 * 2.0 ** -24 + 1e-9
        assert ((m[e].double() - m1[e]).abs() <= 4 * 2.0 ** -24 * (m[e].double().abs() + m1[e].abs() + grad[e].double().abs())).all()


def test_streams_and_graph(dev):
    from mintext_amd.kernels import newton_schulz

    x, y = (torch.stack([gradient(65, 130, r)] * 3).to(dev) for r in (5, 200))
    want, want_y = newton_schulz(x), newton_schulz(y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = newton_schulz(y)
    here = newton_schulz(x)  # at the same time
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(here, want) and torch.equal(other, want_y)
    held = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = newton_schulz(held)
    for t, w in ((x, want), (y, want_y), (x, want)):
        held.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w) and torch.equal(newton_schulz(t), w)
