"""``newton_schulz`` and ``muon_update`` where something is watching that they cannot serve (host only)."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from mintext_amd.kernels import muon_update, newton_schulz

NAMES = ["newton_schulz", "grad", "param", "momentum", "lr"]


def call(name, t):
    """The op with ``t`` as the operand ``name``."""
    if name == "newton_schulz":
        return newton_schulz(t)
    operands = {"param": torch.randn(3, 4, 8), "grad": torch.randn(3, 4, 8), "momentum": torch.zeros(3, 4, 8), "lr": 0.1}
    operands[name] = t
    return muon_update(operands["param"], operands["grad"], operands["momentum"], lr=operands["lr"])


def operand(name):
    return torch.tensor([0.1]) if name == "lr" else torch.randn(3, 4, 8)


@pytest.mark.parametrize("name", NAMES)
def test_a_tangent_is_refused(name):
    with forward_ad.dual_level():
        t = operand(name)
        dual = forward_ad.make_dual(t, torch.ones_like(t))
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(name, dual)
        for plain in (t.clone(), dual.detach()):  # accepted up to the device
            with pytest.raises(RuntimeError, match="GPU tensor"):
                call(name, plain)


@pytest.mark.parametrize("name", NAMES)
def test_a_trace_is_refused(name):
    with pytest.raises(RuntimeError, match="jit trace"):
        torch.jit.trace(lambda t: call(name, t), operand(name), check_trace=False)
