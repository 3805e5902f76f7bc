"""The end of a training step together: experts or a dense layer, the norm behind its residual, the head's loss and a teacher's,
their gradients, and the optimiser's step."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

V_ = 2.0 ** -24


def inputs(dev, T, D, V, K, dtype):
    g = torch.Generator(device=dev).manual_seed(11)
    n = lambda *s, std=1.0: (torch.randn(*s, device=dev, generator=g) * std).to(dtype)
    p = dict(x=n(T, D), w1=n(D, D, std=D ** -0.5), scale=1 + n(D, std=0.1), shift=n(D, std=0.1), table=n(V, D, std=1.5 * D ** -0.5))
    y = torch.randint(0, V, (T,), device=dev, generator=g)
    y[::7] = -100
    idx = torch.randint(0, V, (T, K), device=dev, generator=g)
    idx[::5, K // 2:] = -1
    return p, y, idx, torch.randn(T, K, device=dev, generator=g)


def loss_of(p, y, idx, t, rms):
    from mintext_amd.kernels import layer_norm, linear, linear_cross_entropy, linear_distillation, rms_norm

    a = linear(p["x"], p["w1"], activation="silu")
    h, s = rms_norm(a, p["scale"], residual=p["x"]) if rms else layer_norm(a, p["scale"], p["shift"], residual=p["x"])
    head = p["table"].t()
    ce = linear_cross_entropy(h, head, y, z_loss=1e-3)
    kd = linear_distillation(h, head, idx, t, temperature=2.0)
    return 0.5 * ce + 0.5 * kd + 1e-2 * s.square().mean(dtype=torch.float32)


def loss64(p, y, idx, t, rms):
    f = torch.nn.functional
    s = f.silu(p["x"] @ p["w1"]) + p["x"]
    d = s if rms else s - s.mean(1, keepdim=True)
    h = d / (d.square().mean(1, keepdim=True) + (1e-6 if rms else 1e-5)).sqrt() * p["scale"] + (0 if rms else p["shift"])
    z = h @ p["table"].t()
    live = y >= 0
    lse = torch.logsumexp(z, 1)
    ce = (f.cross_entropy(z, y, reduction="none") + 1e-3 * lse ** 2)[live].mean()
    on = idx >= 0
    q = torch.softmax(torch.where(on, t.double() / 2, -torch.inf), 1)
    lq = torch.log_softmax(z / 2, 1).gather(1, idx.clamp(min=0))
    kd = 4 * torch.where(on, q * (torch.log(q.clamp(min=1e-300)) - lq), 0.0).sum(1).mean()
    return 0.5 * ce + 0.5 * kd + 1e-2 * s.square().mean()


@pytest.mark.parametrize("rms", [True, False])
def test_gradients_through_all_of_them(dev, rms):
    """In float32: reductions of D, D, V and T terms follow each other, each off by at most as many half steps of its terms' sizes,
    which are at most 8 times the results' 2-norms here; the table is used twice."""
    T, D, V, K = 45, 64, 700, 6
    p, y, idx, t = inputs(dev, T, D, V, K, torch.float32)
    names = [k for k in p if k != "shift" or not rms]
    for k in names:
        p[k].requires_grad_(True)
    loss = loss_of(p, y, idx, t, rms)
    grads = torch.autograd.grad(loss, [p[k] for k in names])
    q = {k: v.detach().double().requires_grad_(True) for k, v in p.items()}
    want = loss64(q, y, idx, t, rms)
    assert (loss.detach().double() - want.detach()).abs() <= 8 * (2 * D + V) * V_ * want.detach().abs()
    for k, a, b in zip(names, grads, torch.autograd.grad(want, [q[k] for k in names])):
        assert (a.double() - b).norm() <= 8 * (2 * D + V + T) * V_ * b.norm(), k


def test_training_steps(dev):
    """Three steps with the experts in bfloat16: they run, every gradient is finite, a repeated step gives the same bits."""
    from mintext_amd.kernels import linear_cross_entropy, linear_distillation, muon_update, rms_norm
    from mintext_amd.moe import moe_block_forward

    T, D, V, K, E, inner = 130, 128, 1000, 5, 8, 64
    t = torch.bfloat16
    p, y, idx, tl = inputs(dev, T, D, V, K, t)
    g = torch.Generator(device=dev).manual_seed(3)
    n = lambda *s, std: (torch.randn(*s, device=dev, generator=g) * std).to(t)
    start = dict(gate=n(D, E, std=D ** -0.5), up=n(E, D, 2 * inner, std=D ** -0.5), down=n(E, inner, D, std=inner ** -0.5),
                 table=p["table"], scale=p["scale"].float())

    def run(steps):
        w = {k: v.clone().requires_grad_(True) for k, v in start.items()}
        momentum = {k: torch.zeros_like(w[k], dtype=torch.float32) for k in ("up", "down")}
        out = []
        for _ in range(steps):
            a, _ = moe_block_forward(p["x"], w["gate"], w["up"], w["down"], k=2, scoring="softmax")
            h, _ = rms_norm(a.to(t), w["scale"], residual=p["x"])
            loss = linear_cross_entropy(h, w["table"].t(), y) + linear_distillation(h, w["table"].t(), idx, tl)
            grads = dict(zip(w, torch.autograd.grad(loss, list(w.values()))))
            assert torch.isfinite(loss) and all(torch.isfinite(v).all() and v.any() for v in grads.values())
            assert grads["table"].shape == (V, D) and grads["scale"].dtype == torch.float32
            with torch.no_grad():
                for k in momentum:
                    muon_update(w[k], grads[k], momentum[k], lr=0.02)
                for k in ("gate", "table", "scale"):
                    w[k] -= 0.1 * grads[k]
            out += [loss.detach()] + [grads[k] for k in w]
        return out

    for a, b in zip(run(3), run(3)):
        assert torch.equal(a, b)
