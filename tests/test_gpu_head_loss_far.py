"""The head's losses where logits are far from zero, or some are infinite, against the formulas in 64 bits.

The logits here are exact in float32: x is [b, a, 0, ..], a class's weight [c, n, 0, ..] with b c = base, a = j / 4 and n = i / 64, so
that z = base + i j / 256, of 21 bits at most, as is every partial sum.  What softmax has to do with is then the distance
far = (max z - z) / tau alone.  With v the half step of float32:
  el = sum q 16 v (1 + far) + v (V / 64 + 64)         the logarithm of the sum: each term's exponent, the sum over blocks and lanes
  es = v ((K + 16) (1 + (max t - t) / tau))           a share, relative to it
  L  : tau^2 (el + sum p ((K + 16) v (|log p| + far) + es (1 + |log p| + far)) + 4 v |log sum|) + 4 v |L|
  ed = |g| tau (q (16 v (1 + far) + el) + (es + 16 v) share) + 4 v |dz|    dz before it is rounded (half: what that takes of it)
  dx : u |dx| + (ed + half |dz|) |W|^T + (V + 8) v |dz| |W|^T;  dW: alike with T terms
What lies below the least normal number, 2^-126, may be taken as 0: an exponential (the front factor times that of dz), dz itself, a
product or a result (each once).
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

V_, LEAST = 2.0 ** -24, 2.0 ** -126
BF, F32 = torch.bfloat16, torch.float32


def close(got, want, tol, what):
    assert got.shape == want.shape, what
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float((off / tol)[bad].max()):.2f} x"


# few rows (dz in two planes); small tiles; more of them; large tiles
SIZES = [(3, 1000), (64, 2056), (130, 1000), (300, 2050), (2048, 6400)]


@pytest.mark.parametrize("kind", ["ce", "kd"])
@pytest.mark.parametrize("order", ["dv", "vd"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,V", SIZES)
def test_logits_far_from_zero(dev, T, V, dtype, order, kind):
    from mintext_amd.kernels import linear_cross_entropy, linear_distillation

    K, tau = (1, 1.0) if kind == "ce" else (6, 0.01)
    b, c = (64.0, 64.0) if kind == "ce" else (8.0, 4.0)  # logits around 4096, or around 32 at a temperature of 0.01
    gen = torch.Generator(device=dev).manual_seed(T + V)
    j = torch.randint(1, 5, (T,), device=dev, generator=gen) * torch.where(torch.rand(T, device=dev, generator=gen) < 0.5, 1, -1)
    i = torch.randint(-255, 256, (V,), device=dev, generator=gen)
    x, w = torch.zeros(T, 8, device=dev), torch.zeros(8, V, device=dev)
    x[:, 0], x[:, 1], w[0], w[1] = b, j / 4, c, i / 64
    x, w = x.to(dtype), w.to(dtype)
    w = w.t().contiguous().t() if order == "vd" else w
    z = torch.mm(x.double(), w.double())
    assert torch.equal(z, z.float().double())
    g = torch.rand(T, device=dev, generator=gen) + 0.5

    k = 1 / tau
    far = (z.amax(1, keepdim=True) - z) * k
    near = torch.topk(z, K, 1).indices  # the named classes are among those that count
    if kind == "ce":
        near = torch.where(torch.rand(T, 1, device=dev, generator=gen) < 0.5, near, torch.randint(0, V, (T, 1), device=dev, generator=gen))
        p, es = torch.ones(T, 1, device=dev).double(), torch.zeros(T, 1, device=dev).double()
        call = lambda a, h, r: linear_cross_entropy(a, h, near[:, 0], reduction=r)
    else:
        t = torch.randn(T, K, device=dev, generator=gen) * 0.02
        p = torch.softmax(t.double() * k, 1)
        es = V_ * (K + 16) * (1 + (t.amax(1, keepdim=True) - t).double() * k)
        call = lambda a, h, r: linear_distillation(a, h, near, t, temperature=tau, reduction=r)
    lp = torch.where(p > 0, torch.log(p.clamp(min=1e-300)), 0.0)
    share, sharing = (torch.zeros(T, V, device=dev).double().scatter_add_(1, near, v) for v in (p, p * (es + 16 * V_)))
    q = torch.softmax(z * k, 1)
    log_sum = torch.log(torch.exp(-far).sum(1))
    el = (q * 16 * V_ * (1 + far)).sum(1) + V_ * (V / 64 + 64)
    at = far.gather(1, near)
    want = tau ** 2 * ((p * (lp + at)).sum(1) + log_sum)
    tol = tau ** 2 * (el + (p * ((K + 16) * V_ * (lp.abs() + at) + es * (1 + lp.abs() + at))).sum(1) + 4 * V_ * log_sum.abs())
    loss = call(x.requires_grad_(True), w.requires_grad_(True), "none")
    close(loss.detach(), want, tol + 4 * V_ * want.abs(), "loss")

    unit = (g.double() * tau)[:, None]
    dz = unit * (q - share)
    u = torch.finfo(dtype).eps / 2
    half = u * u if dtype is BF and T <= 64 else u
    er = unit * (q * (16 * V_ * (1 + far) + el[:, None]) + sharing) + (half + 4 * V_) * dz.abs()
    er = er + LEAST * (1 + unit)
    X, W = x.detach().double(), w.detach().double().contiguous()
    gx, gw = torch.autograd.grad(loss, [x, w], g)
    dx, dw = torch.mm(dz, W.t()), torch.mm(X.t(), dz)
    close(gx, dx, u * dx.abs() + torch.mm(er + (V + 8) * V_ * dz.abs(), W.abs().t().contiguous()) + LEAST * (V + 1), "dx")
    close(gw, dw, u * dw.abs() + torch.mm(X.abs().t().contiguous(), er + (2 * T + 8) * V_ * dz.abs()) + LEAST * (T + 1), "dw")


@pytest.mark.parametrize("order", ["dv", "vd"])
@pytest.mark.parametrize("T,D,V", [(20, 33, 301), (20, 31, 304), (64, 1, 300), (130, 39, 301), (300, 65, 512), (2048, 97, 6401)])
def test_weight_of_minus_infinity_takes_a_class_out(dev, T, D, V, order):
    """A weight of -inf in the last row, where the row's x are positive: the class's logit is -inf, its probability 0.  The losses and
    the gradients are those without it, but for that row's share of dx, 0 times -inf.  Widths end a stage or 1 to 7 before an
    eight; the bounds are the logits' (D + 2) v |x| |W|, twice, with those at the file's head for logits of 16 at most."""
    from mintext_amd.kernels import linear_cross_entropy

    gen = torch.Generator(device=dev).manual_seed(T + D)
    x = torch.randn(T, D, device=dev, generator=gen)
    x[:, -1] = x[:, -1].abs() + 0.5
    x = x.to(BF)
    w = (torch.randn(D, V, device=dev, generator=gen) * D ** -0.5).to(BF)
    w[-1, 0] = -float("inf")
    w = w.t().contiguous().t() if order == "vd" else w
    y = torch.randint(1, V, (T,), device=dev, generator=gen)
    X, W = x.double(), w[:, 1:].double()
    z = torch.mm(X, W)
    assert z.abs().max() <= 16
    ez = (D + 2) * V_ * torch.mm(X.abs(), W.abs())
    lse = torch.logsumexp(z, 1)
    want = lse - z.gather(1, y[:, None] - 1)[:, 0]
    el = ez.amax(1) + V_ * (16 * 33 + V / 64 + 64)
    loss = linear_cross_entropy(x.requires_grad_(True), w.requires_grad_(True), y, reduction="none")
    close(loss.detach(), want, 2 * el + 8 * V_ * (16 + want), "loss")
    gx, gw = torch.autograd.grad(loss, [x, w], torch.ones(T, device=dev))
    q = torch.softmax(z, 1)
    dz = q.scatter_add(1, y[:, None] - 1, -torch.ones(T, 1, device=dev).double())
    u = 2.0 ** -8
    er = q * (ez + el[:, None] + 16 * V_ * 33) + 32 * V_ + (u + 4 * V_) * dz.abs()
    dx, dw = torch.mm(dz, W.t()), torch.mm(X.t(), dz)
    tx = u * dx.abs() + torch.mm(er + (V + 8) * V_ * dz.abs(), W.abs().t().contiguous())
    close(gx[:, :-1], dx[:, :-1], tx[:, :-1], "dx")
    close(gw[:, 1:], dw, u * dw.abs() + torch.mm(X.abs().t().contiguous(), er + (2 * T + 8) * V_ * dz.abs()), "dw")
    assert not gw[:, 0].any()


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("T", [5, 70])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_teacher_logit_without_a_softmax(dev, dtype, T, value):
    """An entry of +inf leaves a token no softmax, as one of NaN does: its loss and its whole gradient are NaN, the weight's too,
    and no other token's.  In an empty place it is not looked at."""
    from mintext_amd.kernels import linear_distillation

    gen = torch.Generator(device=dev).manual_seed(T)
    x = torch.randn(T, 40, device=dev, generator=gen).to(dtype).requires_grad_(True)
    w = (torch.randn(40, 300, device=dev, generator=gen) * 0.1).to(dtype).requires_grad_(True)
    idx = torch.randint(0, 300, (T, 3), device=dev, generator=gen)
    idx[1, 2] = -1
    t = torch.randn(T, 3, device=dev, generator=gen)
    clean = linear_distillation(x, w, idx, t, reduction="none")
    (cx,) = torch.autograd.grad(clean.sum(), [x])
    t[1, 2] = value
    assert torch.equal(linear_distillation(x, w, idx, t, reduction="none"), clean)
    t[2, 0] = value
    loss = linear_distillation(x, w, idx, t, reduction="none")
    gx, gw = torch.autograd.grad(loss.sum(), [x, w])
    keep = torch.arange(T, device=dev) != 2
    assert torch.isnan(loss[2]) and torch.isnan(gx[2]).all() and torch.isnan(gw).all()
    assert torch.equal(loss[keep], clean[keep]) and torch.equal(gx[keep], cx[keep])
