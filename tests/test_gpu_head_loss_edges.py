"""Calls of the head's losses at the ends of what they admit: the most tokens, temperatures of 1e-3 and 1e3, operands that are one
tensor, two streams and two threads at once."""
from __future__ import annotations

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

V_ = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("order", ["dv", "vd"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_most_tokens(dev, dtype, order):
    """65535 * 64 tokens, the gradients in pieces of 256 columns.  Losses and dx of rows all along, dW of all: with logits of at most 12
    and |x| |W| of at most 40 a logit is off by 10 v 40, a loss by twice that and 64 v, q alike; dz by half a step u of itself more.
    dW: runs of T / 16 products at most and 16 of them, of what is off by that."""
    from mintext_amd.kernels import linear_cross_entropy

    T, D, V = 65535 * 64, 8, 300
    gen = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn(T, D, device=dev, generator=gen).clamp(-4, 4).to(dtype)
    w = (torch.randn(D, V, device=dev, generator=gen) * 0.3).clamp(-1, 1).to(dtype)
    w = w.t().contiguous().t() if order == "vd" else w
    y = torch.randint(0, V, (T,), device=dev, generator=gen, dtype=torch.int32)
    y[torch.rand(T, device=dev, generator=gen) < 0.1] = -100
    g = torch.rand(T, device=dev, generator=gen) + 0.5
    x.requires_grad_(True), w.requires_grad_(True)
    loss = linear_cross_entropy(x, w, y, reduction="none")
    gx, gw = torch.autograd.grad(loss, [x, w], g)
    W = w.detach().double().contiguous()
    u, e = torch.finfo(dtype).eps / 2, (2 * 10 * 40 + 64) * V_
    dw = torch.zeros(D, V, device=dev, dtype=torch.float64)
    tw = torch.zeros_like(dw)
    for i in range(0, T, 1 << 18):
        X, t = x.detach()[i:i + (1 << 18)].double(), y[i:i + (1 << 18)].long()
        live = (t >= 0).double()[:, None]
        z = torch.mm(X, W)
        assert z.abs().max() <= 12
        lse = torch.logsumexp(z, 1)
        want = (lse - z.gather(1, t.clamp(min=0)[:, None])[:, 0]) * live[:, 0]
        assert ((loss.detach()[i:i + (1 << 18)].double() - want).abs() <= 2 * e + 8 * V_ * want).all()
        q = torch.exp(z - lse[:, None]) * live
        dz = q.scatter_add(1, t.clamp(min=0)[:, None], -live) * g[i:i + (1 << 18)].double()[:, None]
        er = u * dz.abs() + 1.5 * (2 * e * q + 32 * V_ * live)
        dx = torch.mm(dz, W.t())
        tx = u * dx.abs() + torch.mm(er + (V + 8) * V_ * dz.abs(), W.abs().t().contiguous())
        assert ((gx[i:i + (1 << 18)].double() - dx).abs() <= tx).all()
        dw += torch.mm(X.t(), dz)
        tw += torch.mm(X.abs().t().contiguous(), er + (T / 16 + 32) * V_ * dz.abs())
    assert ((gw.double() - dw).abs() <= u * dw.abs() + tw).all()
    # what is off is by far not all of one sign
    assert (gw.double() - dw).norm() <= (0.01 if dtype is BF else 1e-3) * dw.norm()


@pytest.mark.parametrize("T", [9, 200])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_ends_of_the_temperature(dev, dtype, T):
    """1e-3: softmax is the largest logit's (logits are multiples of 1 / 4 up to 8, all exact), and 1e3: it is all but even."""
    from mintext_amd.kernels import linear_distillation

    gen = torch.Generator(device=dev).manual_seed(T)
    V, K = 500, 4
    x = torch.randint(-2, 3, (T, 8), device=dev, generator=gen).to(dtype).requires_grad_(True)
    w = (torch.randint(-2, 3, (8, V), device=dev, generator=gen) / 4).to(dtype).requires_grad_(True)
    z = torch.mm(x.detach().double(), w.detach().double())
    idx = torch.topk(z, K, 1).indices
    t = torch.randint(0, 3, (T, K), device=dev, generator=gen).float()
    for tau in (1e-3, 1e3):
        k = 1 / tau
        p = torch.softmax(t.double() * k, 1)
        q = torch.softmax(z * k, 1)
        lq = torch.log_softmax(z * k, 1).gather(1, idx)
        want = tau ** 2 * (torch.where(p > 0, p * (torch.log(p.clamp(min=1e-300)) - lq), 0.0)).sum(1)
        loss = linear_distillation(x, w, idx, t, temperature=tau, reduction="none")
        # each of the terms is off by some roundings of itself: exponents up to 8 / tau, logarithms of up to log V
        size = tau ** 2 * (1 + torch.log(torch.tensor(float(V))) + (p * lq.abs()).sum(1) + 20 * V_ * 16 * k)
        assert ((loss.detach().double() - want).abs() <= 40 * V_ * size).all()
        gx, gw = torch.autograd.grad(loss.sum(), [x, w])
        dz = tau * q.scatter_add(1, idx, -p)
        u = torch.finfo(dtype).eps / 2
        half = u * u if dtype is BF and T <= 64 else u
        er = (half + 8 * V_) * dz.abs() + tau * V_ * ((64 + 16 * 16 * k) * q + 64 * torch.zeros_like(q).scatter_add(1, idx, p))
        dx, dw = torch.mm(dz, w.detach().double().t()), torch.mm(x.detach().double().t(), dz)
        tx = torch.mm(er + (V + 8) * V_ * dz.abs(), w.detach().double().abs().t().contiguous()) + 2.0 ** -100
        tw = torch.mm(x.detach().double().abs().t().contiguous(), er + (2 * T + 8) * V_ * dz.abs()) + 2.0 ** -100
        assert ((gx.double() - dx).abs() <= u * dx.abs() + tx).all()
        assert ((gw.double() - dw).abs() <= u * dw.abs() + tw).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_operands_that_are_one_tensor(dev, dtype):
    """x against itself: the gradient is the sum of both, as two leaves have it, rounded once more."""
    from mintext_amd.kernels import layer_norm, linear_cross_entropy

    x = torch.randn(96, 64, device=dev).to(dtype).requires_grad_(True)
    a, b = x.detach().clone().requires_grad_(True), x.detach().clone().requires_grad_(True)
    y = torch.arange(96, device=dev)
    (g,) = torch.autograd.grad(linear_cross_entropy(x, x.t(), y), [x])
    ga, gb = torch.autograd.grad(linear_cross_entropy(a, b.t(), y), [a, b])
    assert torch.equal(g, ga + gb)
    w, c = torch.randn(64, device=dev), torch.randn(64, device=dev)
    grads = lambda r, leaves: torch.autograd.grad([*layer_norm(leaves[0], w, c, residual=r)], leaves, [x.detach(), x.detach() * 2])
    (g,), (ga, gb) = grads(x, [x]), grads(b, [a, b])
    assert torch.equal(ga, gb) and torch.equal(g, ga + gb)
    # gradients that are one tensor inside are the caller's to change, each by itself
    a.grad = b.grad = None
    out, h = layer_norm(a, w, c, residual=b)
    (out.float().sum() + h.float().sum()).backward()
    assert torch.equal(a.grad, b.grad) and a.grad.data_ptr() != b.grad.data_ptr()


def test_two_streams_and_threads_at_once(dev):
    """Steps of two sizes on two streams, from two threads, each as it is alone."""
    from mintext_amd.kernels import layer_norm, linear_cross_entropy, linear_distillation

    def make(T, D, V, seed):
        gen = torch.Generator(device=dev).manual_seed(seed)
        x, w = torch.randn(T, D, device=dev, generator=gen).to(BF), (torch.randn(D, V, device=dev, generator=gen) * D ** -0.5).to(BF)
        s = torch.rand(D, device=dev, generator=gen).to(BF)
        y = torch.randint(0, V, (T,), device=dev, generator=gen)
        idx, t = torch.randint(0, V, (T, 9), device=dev, generator=gen), torch.randn(T, 9, device=dev, generator=gen)

        def step():
            leaves = [v.detach().requires_grad_(True) for v in (x, w, s)]
            h = layer_norm(leaves[0], leaves[2])
            loss = linear_cross_entropy(h, leaves[1], y) + linear_distillation(h, leaves[1], idx, t, temperature=2.0)
            return [loss.detach()] + list(torch.autograd.grad(loss, leaves))
        return step

    steps = [make(700, 256, 4104, 1), make(61, 136, 2003, 2)]
    want = [s() for s in steps]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[i].append(steps[i]())
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 - handed to the test
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join(60) for t in threads]
    assert not errors and [len(g) for g in got] == [10, 10]
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
