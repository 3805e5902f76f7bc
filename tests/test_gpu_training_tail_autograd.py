"""What autograd, its transforms and traces see of the norms and the head's losses: second derivatives, vmap, torch.func.grad and
forward-mode tangents are refused, and a trace holds for other numbers of tokens."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

OPS = ["layer_norm", "layer_norm_residual", "rms_norm", "linear_cross_entropy", "linear_distillation"]


def build(dev, op, T=10, D=64, V=90):
    """The operator as a function of x, and x; of one tensor out."""
    from mintext_amd import kernels as k

    g = torch.Generator(device=dev).manual_seed(1)
    x, w, b = (torch.randn(*s, device=dev, generator=g) for s in ((T, D), (D,), (D,)))
    head = torch.randn(D, V, device=dev, generator=g) * 0.1
    # classes and teachers of a token follow from its x, so that a call with other tokens has its own
    classes = lambda a: (a.detach()[..., :1].abs() * 1000).long() % V
    return {
        "layer_norm": lambda a: k.layer_norm(a, w, b),
        "layer_norm_residual": lambda a: k.layer_norm(a, w, b, residual=a.detach() * 0.5)[0],
        "rms_norm": lambda a: k.rms_norm(a, w),
        "linear_cross_entropy": lambda a: k.linear_cross_entropy(a, head, classes(a)[..., 0], reduction="none"),
        "linear_distillation": lambda a: k.linear_distillation(a, head, classes(a), a.detach()[..., :1].contiguous(), reduction="none"),
    }[op], x


@pytest.mark.parametrize("op", OPS)
def test_second_derivative_is_refused(dev, op):
    f, x = build(dev, op)
    x.requires_grad_(True)
    (plain,) = torch.autograd.grad(f(x).sum(), [x])
    (g,) = torch.autograd.grad(f(x).sum(), [x], create_graph=True)
    assert torch.equal(plain, g)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), [x])


@pytest.mark.parametrize("op", OPS)
def test_transforms_are_refused(dev, op):
    f, x = build(dev, op)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda a: f(a).sum())(x)
    with pytest.raises(RuntimeError):
        torch.func.vmap(f)(x)
    with pytest.raises(RuntimeError):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(RuntimeError):
        f(fwd.make_dual(x, torch.ones_like(x)))
    assert torch.isfinite(f(x)).all()  # and leave the operator as it was


@pytest.mark.parametrize("op", ["layer_norm", "layer_norm_residual", "rms_norm"])
def test_trace_holds_for_other_sizes(dev, op):
    f, x = build(dev, op)
    other = torch.randn(23, 64, device=dev)
    with torch.no_grad():
        assert torch.equal(torch.jit.trace(f, (x,), check_trace=False)(other), f(other))
