"""How far the bf16 gradients of the head's losses are off as a whole.

A rounding to half steps of u = 2^-8 relative to a value is off by u |value| / sqrt(3) in the root of its mean square where the
values lie evenly between two steps, and by less where they lie far from the lower power of two.  Roundings of many values are
independent, so the squares of what they leave in a sum add up:
  ||error of dx||^2 <= sum (u |dx|)^2 / 3 + sum ((u |dz|)^2 / 3) (W^2)^T       dW: alike, of x
where dz is rounded once (more than 64 tokens); with the second plane of dz its share is u times as large.  What float32 adds is
below 2^-12 of either.  Twice the loss of a single rounding would not pass.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -8


@pytest.mark.parametrize("kind", ["ce", "kd"])
@pytest.mark.parametrize("order", ["dv", "vd"])
@pytest.mark.parametrize("T,D,V", [(16, 1024, 4096), (64, 520, 5003), (65, 1024, 4096), (300, 520, 5003), (1500, 264, 8200), (4099, 256, 4104)])
def test_norm_of_the_gradients_errors(dev, T, D, V, order, kind):
    from mintext_amd.kernels import linear_cross_entropy, linear_distillation

    gen = torch.Generator(device=dev).manual_seed(T + D + V)
    x = torch.randn(T, D, device=dev, generator=gen).bfloat16()
    w = (torch.randn(V, D, device=dev, generator=gen) * (1.5 * D ** -0.5)).bfloat16()
    w = w.t() if order == "vd" else w.t().contiguous()
    g = torch.rand(T, device=dev, generator=gen) + 0.5
    K = 1 if kind == "ce" else 8
    idx = torch.stack([torch.randperm(V, device=dev, generator=gen)[:K] for _ in range(T)])
    t = torch.randn(T, K, device=dev, generator=gen)
    X, W = x.double(), w.double().contiguous()
    z = torch.mm(X, W)
    dz = torch.softmax(z, 1).scatter_add(1, idx, -torch.softmax(t.double(), 1)) * g.double()[:, None]
    dx, dw = torch.mm(dz, W.t()), torch.mm(X.t(), dz)
    x.requires_grad_(True), w.requires_grad_(True)
    loss = (linear_cross_entropy(x, w, idx[:, 0], reduction="none") if kind == "ce" else
            linear_distillation(x, w, idx, t, reduction="none"))
    gx, gw = torch.autograd.grad(loss, [x, w], g)
    left = (U * dz * (U if T <= 64 else 1)) ** 2 / 3
    for got, want, moved in ((gx, dx, torch.mm(left, W.t() ** 2)), (gw, dw, torch.mm(X.t() ** 2, left))):
        bound = torch.sqrt(((U * want) ** 2 / 3 + moved).sum()) + 2.0 ** -12 * want.norm()
        off = (got.double() - want).norm()
        assert off <= bound, f"{float(off / want.norm()):.2e} off, bound {float(bound / want.norm()):.2e}"
